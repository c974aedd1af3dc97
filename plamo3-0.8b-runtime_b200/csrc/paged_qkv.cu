// QK-norm, rotary embedding and paged cache append of a step's projection rows (plamo_k_paged_qkv).
//
//   y = x * rsqrt(mean(x^2) + eps) * (1 + w);  (y_d, y_{d + D/2}) turned by the position's (cos, sin)
// All in fp32 from the 16-bit inputs, one rounding where a value is stored. (The forward's own k_qkv
// rounds between the operations, as the reference does; the paged step has no reference to follow.)
//
// A head of D 16-bit values is D/8 lanes of 16 bytes; neighbouring lane groups take neighbouring heads of
// a token, so a warp reads 512 consecutive bytes. The mean is a shuffle tree in the group, the rotation's
// other half comes from the lane D/16 away. Memory bound for long calls: each row is read and written once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "paged.h"

namespace plamo {
namespace {

constexpr int QKV_THREADS = 256;

template <bool HALF>
__device__ __forceinline__ float2 widen(uint32_t pair) {
    if (HALF) return __half22float2(*reinterpret_cast<const __half2*>(&pair));
    return make_float2(lo_bf(pair), hi_bf(pair));
}
template <bool HALF>
__device__ __forceinline__ uint32_t narrow(float x, float y) {
    if (HALF) {
        const __half2 h = __floats2half2_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __nv_bfloat162 b = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&b);
}

template <int D, bool HALF>
__global__ void __launch_bounds__(QKV_THREADS) k_paged_qkv(PagedQkvArgs a) {
    constexpr int LANES = D / 8;  // lanes of one head
    const int KV = a.cache.kv_heads, heads = a.heads + 2 * KV;
    const long long unit = ((long long)blockIdx.x * QKV_THREADS + threadIdx.x) / LANES;
    const int sub = threadIdx.x % LANES;
    const int token = int(unit / heads), head = int(unit - (long long)token * heads);
    // whole warps reach the shuffles: a lane group past the end works on the last token and stores nothing
    const bool inside = token < a.tokens;
    const int tok = inside ? token : a.tokens - 1;
    const int slot = a.slots[tok], position = a.rope ? a.positions[tok] : 0;
    const bool live = slot >= 0 && slot < (long long)a.cache.pages * a.cache.page_size &&
                      (!a.rope || (position >= 0 && position < a.rope_rows));
    uint4 v = __ldg(reinterpret_cast<const uint4*>(a.qkv + tok * a.qkv_stride + head * D) + sub);
    if (head < a.heads + KV) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        float x[8];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = widen<HALF>(w[i]);
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
        const uint16_t* norm = head < a.heads ? a.q_norm : a.k_norm;
        if (norm) {
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < 8; i++) ss = fmaf(x[i], x[i], ss);
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(FULL_MASK, ss, o);
            const float inv = 1.0f / sqrtf(ss / D + a.eps);
            const uint4 nw = __ldg(reinterpret_cast<const uint4*>(norm) + sub);
            const uint32_t n[4] = {nw.x, nw.y, nw.z, nw.w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float2 f = widen<HALF>(n[i]);
                x[2 * i] = x[2 * i] * inv * (1.0f + f.x);
                x[2 * i + 1] = x[2 * i + 1] * inv * (1.0f + f.y);
            }
        }
        if (a.rope) {
            const uint4* cs4 = reinterpret_cast<const uint4*>(a.rope + (long long)(live ? position : 0) * (D / 2) +
                                                              (sub % (LANES / 2)) * 8);
            const uint4 c0 = __ldg(cs4), c1 = __ldg(cs4 + 1);
            const uint32_t cs[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
            const bool low = sub < LANES / 2;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float other = __shfl_xor_sync(FULL_MASK, x[i], LANES / 2);
                x[i] = fmaf(x[i], lo_bf(cs[i]), (low ? -other : other) * hi_bf(cs[i]));
            }
        }
        v = make_uint4(narrow<HALF>(x[0], x[1]), narrow<HALF>(x[2], x[3]), narrow<HALF>(x[4], x[5]),
                       narrow<HALF>(x[6], x[7]));
    }
    if (!inside) return;
    if (head < a.heads) {
        if (!live) v = make_uint4(0u, 0u, 0u, 0u);
        reinterpret_cast<uint4*>(a.q + token * a.q_stride + head * D)[sub] = v;
    } else if (live) {
        const bool key = head < a.heads + KV;
        const int kvh = head - a.heads - (key ? 0 : KV);
        const int page = slot / a.cache.page_size;
        uint16_t* dst = (key ? a.cache.keys : a.cache.values) + page * a.cache.page_stride +
                        (slot - page * a.cache.page_size) * a.cache.token_stride + kvh * a.cache.head_stride;
        reinterpret_cast<uint4*>(dst)[sub] = v;
    }
}

}  // namespace

cudaError_t launch_paged_qkv(const PagedQkvArgs& a, int head_dim, bool half, cudaStream_t s) {
    const long long threads = (long long)a.tokens * (a.heads + 2 * a.cache.kv_heads) * (head_dim / 8);
    const unsigned blocks = unsigned((threads + QKV_THREADS - 1) / QKV_THREADS);
    if (head_dim == 128) {
        if (half) k_paged_qkv<128, true><<<blocks, QKV_THREADS, 0, s>>>(a);
        else k_paged_qkv<128, false><<<blocks, QKV_THREADS, 0, s>>>(a);
    } else {
        if (half) k_paged_qkv<64, true><<<blocks, QKV_THREADS, 0, s>>>(a);
        else k_paged_qkv<64, false><<<blocks, QKV_THREADS, 0, s>>>(a);
    }
    return cudaGetLastError();
}

}  // namespace plamo
