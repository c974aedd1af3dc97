// Block table and slot map of one serving step from the requests' lengths (plamo_k_paged_plan).
//
// held_r = ceil(len_r / page), need_r = ceil((len_r + add_r) / page) - held_r. With F = free pages + the
// pages of ended requests, request r is granted its pages when need_0 + ... + need_r <= F: three running
// sums over the requests decide everything, and each page and token is then an independent lookup.
//
// Every block repeats the sums over the requests (two 32-bit words a request, from L2) and keeps them in
// shared memory, so no block waits for another; the tokens, granted pages and freed pages are spread
// over the grid. A granted page is found without the free list's new end: stack position p is free_list[p]
// below the old count, else an entry of an ended request's table row, which nothing writes in this call.
// Latency bound: two dependent reads, two block scans, one dependent write.
#include "common.cuh"
#include "paged.h"

#include <algorithm>
#include <climits>

namespace plamo {
namespace {

constexpr int PLAN_THREADS = 256;

// Running sum over the block of one value a thread (exclusive), and the block's total.
__device__ __forceinline__ long long block_scan(long long v, long long* warp_sums, long long& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(FULL_MASK, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();  // the sums of an earlier scan have been read
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    long long before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < PLAN_THREADS / 32; w++) {
        if (w < warp) before += warp_sums[w];
        total += warp_sums[w];
    }
    return before + x - v;
}

// The first row whose running sum (inclusive, non-decreasing) exceeds i.
__device__ __forceinline__ int row_of(const int* upto, int rows, int i) {
    int lo = 0, hi = rows - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (upto[mid] > i) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

__device__ __forceinline__ int saturate(long long v) { return v > INT_MAX ? INT_MAX : int(v); }

__global__ void __launch_bounds__(PLAN_THREADS) k_paged_plan(PagedPlanArgs a) {
    extern __shared__ int plan_smem[];
    int* const end = plan_smem;               // running sum of appended tokens, inclusive
    int* const need_upto = end + a.rows;      // running sum of needed pages, inclusive
    int* const freed_upto = need_upto + a.rows;  // running sum of freed pages, inclusive
    int* const state = freed_upto + a.rows;   // length before the step; -1 - length for a refused request
    __shared__ long long warp_sums[PLAN_THREADS / 32];
    const int t = threadIdx.x, P = a.page_size;
    const int per = (a.rows + PLAN_THREADS - 1) / PLAN_THREADS;
    const int r0 = min(t * per, a.rows), r1 = min(r0 + per, a.rows);
    const long long width = a.table_stride;
    // running sum of the appended tokens
    long long sum = 0, tokens_total;
    for (int r = r0; r < r1; r++) sum += max(a.append[r], 0);
    long long at = block_scan(sum, warp_sums, tokens_total);
    // needed and freed pages
    long long need_sum = 0, freed_sum = 0;
    for (int r = r0; r < r1; r++) {
        const int add = a.append[r], len = max(a.lens[r], 0);
        const long long held = min((long long)(len + (long long)P - 1) / P, width);
        const long long want = (long long)len + max(add, 0);
        if (blockIdx.x == 0) a.row_start[r] = saturate(at);
        at += max(add, 0);
        end[r] = saturate(at);
        const bool fits = add >= 0 && want <= width * P && at <= a.tokens;
        const long long need = fits ? (want + P - 1) / P - held : 0;
        need_sum += need;
        freed_sum += add < 0 ? held : 0;
        need_upto[r] = saturate(need);
        freed_upto[r] = add < 0 ? int(held) : 0;
        state[r] = fits || add < 0 ? len : -1 - len;
    }
    long long need_total, freed_total;
    long long need_at = block_scan(need_sum, warp_sums, need_total);
    long long freed_at = block_scan(freed_sum, warp_sums, freed_total);
    const int count0 = min(max(*a.free_count, 0), a.pages);
    const long long F = count0 + freed_total;
    long long granted = 0, refused = 0;
    for (int r = r0; r < r1; r++) {
        const int need = need_upto[r];
        need_at += need;
        freed_at += freed_upto[r];
        need_upto[r] = saturate(need_at);
        freed_upto[r] = saturate(freed_at);
        if (state[r] >= 0 && need > 0 && need_at > F) state[r] = -1 - state[r];
        if (state[r] >= 0) granted += need;
        else refused++;
        if (blockIdx.x == 0) {
            const int add = a.append[r], len = state[r] < 0 ? -1 - state[r] : state[r];
            a.new_lens[r] = add < 0 ? 0 : state[r] < 0 ? len : len + add;
        }
    }
    long long granted_total, refused_total = 0;
    block_scan(granted, warp_sums, granted_total);
    if (blockIdx.x == 0) {
        block_scan(refused, warp_sums, refused_total);
        if (t == 0) {
            a.row_start[a.rows] = saturate(tokens_total);
            a.counts[0] = saturate(F - granted_total);
            a.counts[1] = saturate(tokens_total);
            a.counts[2] = saturate(granted_total);
            a.counts[3] = int(refused_total);
        }
    }
    __syncthreads();  // every row's sums are in shared memory
    // the page at a position of the free stack (its old end first, then the ended requests' pages)
    auto stack_page = [&](long long p) -> int {
        if (p < count0) return a.free_list[p];
        const int i = int(p - count0), r = row_of(freed_upto, a.rows, i);
        const int first = r ? freed_upto[r - 1] : 0;
        return a.table[size_t(r) * a.table_stride + (i - first)];
    };
    const long long stride = (long long)gridDim.x * PLAN_THREADS, id = (long long)blockIdx.x * PLAN_THREADS + t;
    // tokens
    const int live = saturate(min(tokens_total, (long long)a.tokens));
    for (long long i = id; i < a.tokens; i += stride) {
        int slot = -1, position = -1;
        if (i < live) {
            const int r = row_of(end, a.rows, int(i)), len = state[r];
            if (len >= 0) {
                const int start = r ? end[r - 1] : 0;
                position = len + (int(i) - start);
                const int held = (len + P - 1) / P, page = position / P;
                const int id_page = page < held ? a.table[size_t(r) * a.table_stride + page]
                                                : stack_page(F - 1 - ((r ? need_upto[r - 1] : 0) + (page - held)));
                if (id_page >= 0 && id_page < a.pages) slot = id_page * P + position % P;
            }
        }
        a.slots[i] = slot;
        a.positions[i] = position;
    }
    // granted pages into the table
    for (long long i = id; i < granted_total; i += stride) {
        const int r = row_of(need_upto, a.rows, int(i));
        const int held = (state[r] + P - 1) / P;
        a.table[size_t(r) * a.table_stride + held + (int(i) - (r ? need_upto[r - 1] : 0))] = stack_page(F - 1 - i);
    }
    // freed pages onto the free list
    for (long long i = id; i < freed_total && count0 + i < a.pages; i += stride) a.free_list[count0 + i] = stack_page(count0 + i);
}

}  // namespace

cudaError_t launch_paged_plan(const PagedPlanArgs& a, cudaStream_t s) {
    const size_t smem = size_t(4) * a.rows * sizeof(int);
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_shared(k_paged_plan, size_t(4) * PAGED_MAX_ROWS * sizeof(int), done);
    if (e != cudaSuccess) return e;
    const long long work = (long long)a.tokens + 64ll * a.rows;
    const int blocks = int(std::clamp((work + 4 * PLAN_THREADS - 1) / (4 * PLAN_THREADS), 1ll, 148ll));
    k_paged_plan<<<blocks, PLAN_THREADS, smem, s>>>(a);
    return cudaGetLastError();
}

}  // namespace plamo
