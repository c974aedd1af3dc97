// Block table and slot map of one serving step from the requests' lengths (plamo_k_paged_plan).
//
// held_r = ceil(len_r / page), need_r = ceil((len_r + add_r) / page) - held_r. With F = free pages + the
// pages of ended requests, request r is granted its pages when need_0 + ... + need_r <= F: three running
// sums over the requests decide everything, and each page and token is then an independent lookup.
// An ended request's pages are those of its first held_r entries that name one: pages given up before are no
// longer its own. Every block counts them itself (nothing is read where no request ends): 0.7 us for 2 of 32 requests
// with 2000 pages each, 1.8 us for 40 of 1000, half of it the reads, which all SMs make of the same lines at once.
//
// Every block repeats the sums over the requests (two 32-bit words a request, from L2) and keeps them in
// shared memory, so no block waits for another; the tokens, granted pages and freed pages are spread
// over the grid as one line of independent pieces. A granted page is found without the free list's new end: stack position p is free_list[p]
// below the old count, else an entry of an ended request's table row, which nothing writes in this call (its place is
// known where the row's pages lie side by side, as behind a window; else the row is counted through).
// Latency bound: a read of the lengths, two block scans, a search, a table read and the writes follow one another.
// (Four neighbouring tokens a thread, with one search and 16-byte writes, measured 10.3 us against 7.3 for a call of
// 1000 prompts: their steps run one after another.) Blocks have 1024 threads where there are more than 256 requests, so that
// a thread adds up few of them.
#include "common.cuh"
#include "paged.h"

#include <algorithm>
#include <climits>

namespace plamo {
namespace {

// Exclusive running sum over the block, in thread order, and the total.
template <int THREADS>
__device__ __forceinline__ long long block_scan(long long v, long long* warp_sums, long long& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(FULL_MASK, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    long long w = lane < THREADS / 32 ? warp_sums[lane] : 0;
#pragma unroll
    for (int o = 1; o < THREADS / 32; o <<= 1) {
        const long long y = __shfl_up_sync(FULL_MASK, w, o);
        if (lane >= o) w += y;
    }
    total = __shfl_sync(FULL_MASK, w, THREADS / 32 - 1);
    const long long before = __shfl_sync(FULL_MASK, w, max(warp - 1, 0));
    return (warp ? before : 0) + x - v;
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
__device__ __forceinline__ int pages_of(int len, int page_size) {
    return int((unsigned(len) + unsigned(page_size - 1)) / unsigned(page_size));
}

constexpr unsigned CHUNK = 512;  // entries of an ended request that a warp reads at a time (256: 0.2 us more)
// An ended request's row is looked through in up to this many pieces, a warp each: few requests leave warps for them.
__host__ __device__ __forceinline__ int most_pieces(int rows) { return rows <= PAGED_MAX_ROWS / 8 ? 8 : 1; }
__device__ __forceinline__ int pieces_of(unsigned held, int most) { return min(int((held + CHUNK - 1) / CHUNK), most); }

template <int THREADS>
__global__ void __launch_bounds__(THREADS) k_paged_plan(PagedPlanArgs a) {
    pdl_enter();
    extern __shared__ int plan_smem[];
    int* const end = plan_smem;               // running sum of appended tokens, inclusive
    int* const need_upto = end + a.rows;      // running sum of needed pages, inclusive
    int* const freed_upto = need_upto + a.rows;  // running sum of freed pages, inclusive
    int* const state = freed_upto + a.rows;   // length before the step; -1 - length for a refused request; of an
                                              // ended one its first page's entry, SCATTERED when they are apart
    int* const first = state + a.rows;        // of ended requests: the first entry that is a page
    int* const work = first + a.rows;         // pieces of ended requests' rows: piece * PAGED_MAX_ROWS + request
    __shared__ long long token_sums[THREADS / 32];
    __shared__ long long page_sums[THREADS / 32];
    __shared__ int granted_total, refused_total, items;
    constexpr int SCATTERED = INT_MAX;
    const int pieces = most_pieces(a.rows);
    const int t = threadIdx.x, P = a.page_size, width = a.table_stride;
    const long long most = min((long long)width * P, (long long)INT_MAX);  // tokens that a table row can hold
    const int per = (a.rows + THREADS - 1) / THREADS;
    const int r0 = min(t * per, a.rows), r1 = min(r0 + per, a.rows);
    const int count0 = min(max(*a.free_count, 0), a.pages);
    if (t == 0) granted_total = refused_total = items = 0;
    __syncthreads();
    // running sum of the appended tokens; for the ended requests' entries (held, in need_upto) a list of work, in any order
    long long sum = 0, tokens_total;
    for (int r = r0; r < r1; r++) {
        const int add = a.append[r], len = max(a.lens[r], 0);
        state[r] = len;
        end[r] = max(add, -1);
        sum += max(add, 0);
        if (add < 0) {
            freed_upto[r] = 0;
            first[r] = INT_MAX;
            const int held = need_upto[r] = min(pages_of(len, P), width);
            const int n = pieces_of(held, pieces), i = n ? atomicAdd(&items, n) : 0;
            for (int piece = 0; piece < n; piece++) work[i + piece] = piece * PAGED_MAX_ROWS + r;
        }
    }
    __syncthreads();
    // the entries of ended requests that are pages: how many, the first and the last (as -1 - entry, in `end`). A warp
    // takes a piece of a request, CHUNK entries at a time; its first reads are in flight during the sum.
    const int warp = t >> 5, lane = t & 31;
    int item = warp, owner = 0, page[CHUNK / 32];
    unsigned chunk = 0, step = 0, held_by = 0;
    auto take = [&] {
        const unsigned entry = work[item];
        owner = int(entry % PAGED_MAX_ROWS);
        held_by = need_upto[owner];
        chunk = entry / PAGED_MAX_ROWS * CHUNK;
        step = unsigned(pieces_of(held_by, pieces)) * CHUNK;
    };
    auto read = [&] {
        const int* const row = a.table + size_t(owner) * width;
        if (chunk + CHUNK <= held_by) {
#pragma unroll
            for (int e = 0; e < CHUNK / 32; e++) page[e] = row[chunk + lane + 32 * e];
        } else if (held_by - chunk <= CHUNK / 4) {  // short rows by few reads: 0.4 us of 40 among 1000 requests
#pragma unroll
            for (int e = 0; e < CHUNK / 32; e++) page[e] = e < CHUNK / 128 ? row[min(chunk + 32 * e + lane, held_by - 1)] : 0;
        } else {  // past the end the last entry again
#pragma unroll
            for (int e = 0; e < CHUNK / 32; e++) page[e] = row[min(chunk + 32 * e + lane, held_by - 1)];
        }
    };
    if (item < items) {
        take();
        read();
    }
    long long at = block_scan<THREADS>(sum, token_sums, tokens_total);
    if (items) {
        while (item < items) {
            int low = int(chunk), high = int(min(chunk + CHUNK, held_by)) - 1, n = high - low + 1;
            unsigned worst = 0;
#pragma unroll
            for (int e = 0; e < CHUNK / 32; e++) worst = max(worst, unsigned(page[e]));
            if (__any_sync(FULL_MASK, worst >= unsigned(a.pages))) {  // else all of them are pages
                n = 0;
                low = INT_MAX;
                high = -1;
#pragma unroll
                for (int e = 0; e < CHUNK / 32; e++) {
                    const unsigned j = chunk + 32 * e + lane;
                    if (j >= held_by || unsigned(page[e]) >= unsigned(a.pages)) continue;
                    n++;
                    low = min(low, int(j));
                    high = int(j);
                }
                n = __reduce_add_sync(FULL_MASK, n);
                low = __reduce_min_sync(FULL_MASK, low);
                high = __reduce_max_sync(FULL_MASK, high);
            }
            if (lane == 0 && n) {
                atomicAdd(freed_upto + owner, n);
                atomicMin(first + owner, low);
                atomicMin(end + owner, -1 - high);
            }
            chunk += step;
            if (chunk >= held_by) {
                item += THREADS / 32;
                if (item >= items) break;
                take();
            }
            read();
        }
        __syncthreads();
    }
    // needed and freed pages: at most rows * table_stride < 2^31 of each
    int need_sum = 0, freed_sum = 0;
    for (int r = r0; r < r1; r++) {
        const int add = end[r], len = state[r];
        const int held = min(pages_of(len, P), width);
        if (blockIdx.x == 0) a.row_start[r] = saturate(at);
        at += max(add, 0);
        end[r] = saturate(at);
        const long long want = (long long)len + max(add, 0);
        const bool fits = add >= 0 && want <= most && at <= a.tokens;
        const int need = fits ? pages_of(int(want), P) - held : 0, freed = add < 0 ? freed_upto[r] : 0;
        if (add < 0) state[r] = -1 - add - first[r] + 1 == freed ? first[r] : SCATTERED;
        need_sum += need;
        freed_sum += freed;
        need_upto[r] = need;
        freed_upto[r] = freed;
        if (!fits && add >= 0) state[r] = -1 - len;
    }
    long long both_total;  // needed pages in the lower half, freed ones in the upper: neither reaches 2^31
    const long long both = block_scan<THREADS>((long long)freed_sum << 32 | need_sum, page_sums, both_total);
    int need_at = int(both & 0xffffffffll), freed_at = int(both >> 32);
    const int freed_total = int(both_total >> 32);
    const long long F = (long long)count0 + freed_total;
    // what is granted is the needed pages up to the last request that still gets its own
    int granted = 0, refused = 0;
    for (int r = r0; r < r1; r++) {
        const int need = need_upto[r];
        need_at += need;
        freed_at += freed_upto[r];
        need_upto[r] = need_at;
        freed_upto[r] = freed_at;
        int len = state[r];
        if (len >= 0 && need > 0) {
            if (need_at > F) state[r] = len = -1 - len;
            else granted = need_at;
        }
        refused += len < 0;
        if (blockIdx.x == 0) {
            const int add = a.append[r];
            a.new_lens[r] = add < 0 ? 0 : len < 0 ? -1 - len : len + add;
        }
    }
    granted = __reduce_max_sync(FULL_MASK, granted);
    refused = __reduce_add_sync(FULL_MASK, refused);
    if ((t & 31) == 0) {
        if (granted) atomicMax(&granted_total, granted);
        if (refused) atomicAdd(&refused_total, refused);
    }
    __syncthreads();  // every row's sums and the totals are in shared memory
    const int taken = granted_total;
    if (blockIdx.x == 0 && t == 0) {
        a.row_start[a.rows] = saturate(tokens_total);
        a.counts[0] = saturate(F - taken);
        a.counts[1] = saturate(tokens_total);
        a.counts[2] = taken;
        a.counts[3] = refused_total;
    }
    // the page at a position of the free stack (its old end first, then the ended requests' pages)
    auto stack_page = [&](long long p) -> int {
        if (p < count0) return a.free_list[p];
        const int i = int(p - count0), r = row_of(freed_upto, a.rows, i);
        const int* const row = a.table + size_t(r) * width;
        int nth = i - (r ? freed_upto[r - 1] : 0);
        if (state[r] != SCATTERED) return row[state[r] + nth];
        for (int j = 0; j < width; j++) {
            const int page = row[j];
            if (page >= 0 && page < a.pages && nth-- == 0) return page;
        }
        return -1;
    };
    const int live = saturate(min(tokens_total, (long long)a.tokens));
    // the slot and position of token i
    auto token = [&](int i) {
        int slot = -1, position = -1;
        const int r = i < live ? row_of(end, a.rows, i) : 0, len = i < live ? state[r] : -1;
        if (len >= 0) {
            position = len + (i - (r ? end[r - 1] : 0));
            const int of = int(unsigned(position) / unsigned(P)), held = pages_of(len, P);
            const int page = of < held ? a.table[size_t(r) * width + of]
                                       : stack_page(F - 1 - ((r ? need_upto[r - 1] : 0) + (of - held)));
            if (page >= 0 && page < a.pages) slot = page * P + (position - of * P);
        }
        a.slots[i] = slot;
        a.positions[i] = position;
    };
    // one line of independent work: tokens, granted pages into the table, freed pages onto the free list
    const long long granted_end = (long long)a.tokens + taken,
                    all = granted_end + min((long long)freed_total, (long long)a.pages - count0);
    for (long long x = (long long)blockIdx.x * THREADS + t; x < all; x += (long long)gridDim.x * THREADS) {
        if (x < a.tokens) {
            token(int(x));
        } else if (x < granted_end) {
            const int i = int(x - a.tokens), r = row_of(need_upto, a.rows, i);
            a.table[size_t(r) * width + pages_of(state[r], P) + (i - (r ? need_upto[r - 1] : 0))] = stack_page(F - 1 - i);
        } else {
            const long long p = count0 + (x - granted_end);
            a.free_list[p] = stack_page(p);
        }
    }
}

template <int THREADS>
cudaError_t launch(const PagedPlanArgs& a, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_shared(k_paged_plan<THREADS>, size_t(6) * PAGED_MAX_ROWS * sizeof(int), done);
    if (e != cudaSuccess) return e;
    // a thread for a token, and for 64 granted or freed pages a request: those are known on the device only
    const long long work = (long long)a.tokens + 64ll * a.rows;
    const int blocks = int(std::clamp((work + THREADS - 1) / THREADS, 1ll, 148ll));
    return pdl_launch(k_paged_plan<THREADS>, dim3(blocks), dim3(THREADS), size_t(5 + most_pieces(a.rows)) * a.rows * sizeof(int), s, a);
}

}  // namespace

cudaError_t launch_paged_plan(const PagedPlanArgs& a, cudaStream_t s) {
    return a.rows > 256 ? launch<1024>(a, s) : launch<256>(a, s);
}

}  // namespace plamo
