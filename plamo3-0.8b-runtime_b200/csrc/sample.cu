// Sampling by temperature, top-k, top-p and min-p from given uniform numbers (plamo_k_sample).
//
//   w_i = floor(2^40 exp((x_i - max x) / T)) as whole numbers, so sums are exact in any order;
//   kept: a run of the order (x descending, index ascending): the first k, of those the shortest run with
//   at least p of their weight, of those the ones with w >= min_p 2^40;
//   id = the lowest kept index whose running weight (in index order) exceeds floor(2^24 u) W / 2^24.
// The kept run is described by a threshold on the order-preserving key of x and by how many of the values
// at the threshold belong to it, so nothing is sorted.
//
// One block a row. The thresholds are found bit by bit, each bit with one pass over the row.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "paged.h"

namespace plamo {
namespace {

constexpr int SAMPLE_THREADS = 1024;
typedef unsigned long long u64;

// The logit at i as fp32: type 0 bf16, 1 fp16, 2 fp32.
template <int TYPE>
__device__ __forceinline__ float logit_at(const void* row, int i) {
    if (TYPE == 2) return static_cast<const float*>(row)[i];
    const uint16_t b = static_cast<const uint16_t*>(row)[i];
    return TYPE == 1 ? __half2float(__ushort_as_half(b)) : bf2f(b);
}

// Order-preserving key of a logit (larger is larger, -0 equals 0); 0 for NaN and -inf, which are never chosen.
__device__ __forceinline__ uint32_t order_key(float x) {
    if (!(x > -INFINITY)) return 0u;
    const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

__device__ __forceinline__ u64 weight(float x, float top, float temperature) {
    if (!(x > -INFINITY)) return 0ull;
    if (x == top) return 1ull << 40;
    const float e = expf(__fdiv_rn(x - top, temperature));
    return e > 0.f ? u64(e * 1099511627776.0f) : 0ull;
}

// fraction * total / 2^24 in whole numbers (fraction <= 2^24, total < 2^62), rounded down or up
__device__ __forceinline__ u64 share(u64 fraction, u64 total, bool up) {
    return fraction * (total >> 24) + ((fraction * (total & 0xffffffull) + (up ? 0xffffffull : 0ull)) >> 24);
}

struct Sums {
    u64 count, weight;
};

__device__ __forceinline__ u64 warp_add(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL_MASK, v, o);
    return v;
}

__device__ __forceinline__ Sums block_add(Sums v, Sums* scratch) {
    v.count = warp_add(v.count);
    v.weight = warp_add(v.weight);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    Sums s = scratch[threadIdx.x & 31];
    s.count = warp_add(s.count);
    s.weight = warp_add(s.weight);
    return s;
}

// Exclusive running sum over the block in thread order; total returned too.
__device__ __forceinline__ u64 block_scan(u64 v, Sums* scratch, u64& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    u64 x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 y = __shfl_up_sync(FULL_MASK, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) scratch[warp].weight = x;
    __syncthreads();
    u64 before = 0;
    total = 0;
    for (int w = 0; w < SAMPLE_THREADS / 32; w++) {
        if (w < warp) before += scratch[w].weight;
        total += scratch[w].weight;
    }
    return before + x - v;
}

template <int TYPE>
__global__ void __launch_bounds__(SAMPLE_THREADS) k_sample(SampleArgs a) {
    __shared__ Sums scratch[SAMPLE_THREADS / 32];
    __shared__ float tops[SAMPLE_THREADS / 32];
    const int r = blockIdx.x, t = threadIdx.x, V = a.vocab;
    const void* row = static_cast<const uint8_t*>(a.logits) + r * a.row_stride * (TYPE == 2 ? 4 : 2);
    float T = a.temperature ? a.temperature[r] : 1.f;
    const bool warm = T > 0.f;
    if (!warm) T = 1.f;
    int k = !warm ? 1 : a.top_k ? a.top_k[r] : 0;
    if (k <= 0 || k > V) k = V;
    const float top_p = a.top_p ? a.top_p[r] : 1.f, min_p = a.min_p ? a.min_p[r] : 0.f;
    const u64 p24 = top_p < 1.f ? u64(rint(fmax(double(top_p), 0.0) * 16777216.0)) : 1ull << 24;
    const u64 least = max(1ull, min_p > 0.f ? u64(ceil(fmin(double(min_p), 1.0) * 1099511627776.0)) : 0ull);
    // largest logit
    float top = -INFINITY;
    for (int i = t; i < V; i += SAMPLE_THREADS) top = fmaxf(top, logit_at<TYPE>(row, i));
    top = warp_max(top);
    if ((t & 31) == 0) tops[t >> 5] = top;
    __syncthreads();
    top = warp_max(tops[t & 31]);
    // count and weight of the keys >= least_key
    auto above = [&](uint32_t least_key) {
        Sums s{0, 0};
        for (int i = t; i < V; i += SAMPLE_THREADS) {
            const float x = logit_at<TYPE>(row, i);
            const uint32_t key = order_key(x);
            if (key && key >= least_key) {
                s.count++;
                s.weight += weight(x, top, T);
            }
        }
        return block_add(s, scratch);
    };
    // kept: keys above `edge`, and the first `ties` (in index order) of those at it
    uint32_t edge = 0;
    u64 ties = 0, run_weight;
    const Sums all = above(1);
    run_weight = all.weight;
    if (u64(k) < all.count) {
        for (uint32_t bit = 1u << 31; bit; bit >>= 1)
            if (above(edge | bit).count >= u64(k)) edge |= bit;
        const Sums over = above(edge + 1);
        ties = k - over.count;
        run_weight = over.weight + ties * weight(key_value(edge), top, T);
    }
    if (p24 < (1ull << 24) && run_weight) {
        const u64 need = max(share(p24, run_weight, true), 1ull);
        uint32_t cut = 0;
        for (uint32_t bit = 1u << 31; bit; bit >>= 1) {
            const uint32_t c = cut | bit;
            if ((c > edge ? above(c).weight : run_weight) >= need) cut = c;
        }
        const Sums over = above(cut + 1);
        const u64 one = weight(key_value(cut), top, T);
        ties = (need - over.weight + one - 1) / one;
        edge = cut;
    }
    // the ids in index order: each thread a contiguous range
    const int per = (V + SAMPLE_THREADS - 1) / SAMPLE_THREADS, i0 = min(t * per, V), i1 = min(i0 + per, V);
    u64 at_edge = 0, unused;
    for (int i = i0; i < i1; i++) at_edge += edge && order_key(logit_at<TYPE>(row, i)) == edge;
    const u64 first_tie = block_scan(at_edge, scratch, unused);
    auto kept_weight = [&](int i, u64& tie) -> u64 {
        const float x = logit_at<TYPE>(row, i);
        const uint32_t key = order_key(x);
        if (!key || key < edge || (key == edge && tie++ >= ties)) return 0ull;
        const u64 w = weight(x, top, T);
        return w >= least ? w : 0ull;
    };
    Sums mine{0, 0};
    u64 tie = first_tie;
    for (int i = i0; i < i1; i++) {
        const u64 w = kept_weight(i, tie);
        mine.count += w != 0;
        mine.weight += w;
    }
    const Sums total = block_add(mine, scratch);
    const float u = a.u[r];
    const u64 m = u > 0.f ? min(u64(fminf(u, 1.f) * 16777216.0f), (1ull << 24) - 1) : 0ull;
    const u64 target = share(m, total.weight, false);
    u64 before = block_scan(mine.weight, scratch, unused);
    if (before <= target && target < before + mine.weight) {
        tie = first_tie;
        for (int i = i0; i < i1; i++) {
            const u64 w = kept_weight(i, tie);
            if (target < before + w) {
                a.ids[r] = i;
                if (a.logprobs) a.logprobs[r] = float(log(double(w) / double(total.weight)));
                break;
            }
            before += w;
        }
    }
    if (t == 0) {
        if (a.kept) a.kept[r] = int(total.count);
        if (!total.weight) {
            a.ids[r] = 0;
            if (a.logprobs) a.logprobs[r] = -INFINITY;
        }
    }
}

}  // namespace

cudaError_t launch_sample(const SampleArgs& a, int dtype, cudaStream_t s) {
    if (dtype == 0) k_sample<0><<<a.rows, SAMPLE_THREADS, 0, s>>>(a);
    else if (dtype == 1) k_sample<1><<<a.rows, SAMPLE_THREADS, 0, s>>>(a);
    else k_sample<2><<<a.rows, SAMPLE_THREADS, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace plamo
