// QK-norm, rotary embedding and paged cache append of a step's projection rows (plamo_k_paged_qkv).
//
//   y = x * rsqrt(mean(x^2) + eps) * (1 + w);  (y_d, y_{d + D/2}) turned by the position's (cos, sin)
// All in fp32 from the 16-bit inputs, one rounding where a value is stored. (The forward's own k_qkv
// rounds between the operations, as the reference does; the paged step has no reference to follow.)
//
// A lane holds four values of a head's first half and the four that they are rotated with, D/2 further: no
// exchange for the rotation, and one 16-byte read of its cosines and sines. A head is D/8 lanes, so a warp takes
// a step of 2 (D = 128) or 4 heads of one token at a time, four steps' reads in flight together; the
// position's cosines and sines and the norm weights serve every step. The mean is a shuffle tree in the
// head's lanes. Arithmetic runs on pairs (fma.rn.f32x2), which halves the instructions that bound a first
// version of this kernel. Each row is read and written once. Long calls: a warp a token. Short calls: a warp
// a step, to spread over the SMs. Calls with and without a rotation are two kernels (one for both: 20.9 us for
// 8191 tokens of 16 + 2 x 4 heads, so 19.9).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "paged.h"

namespace plamo {
namespace {

constexpr int QKV_THREADS = 128;

// Two fp32 values in one 64-bit register, each operation rounded as the single one is.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair(float x, float y) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 unpair(f32x2 p) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
    return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

template <bool HALF>
__device__ __forceinline__ f32x2 widen(uint32_t two) {
    if (HALF) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&two));
        return pair(f.x, f.y);
    }
    return pair(lo_bf(two), hi_bf(two));
}
template <bool HALF>
__device__ __forceinline__ uint32_t narrow(f32x2 p) {
    const float2 f = unpair(p);
    if (HALF) {
        const __half2 h = __floats2half2_rn(f.x, f.y);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __nv_bfloat162 b = __floats2bfloat162_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t*>(&b);
}

// 8 bytes that are read once: not kept in L1.
__device__ __forceinline__ uint2 read_once(const void* p) {
    uint2 v;
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}

// Steps of a token: its query heads, then its key heads, then its value heads, 256 / D heads a step.
struct Steps {
    int q, kv;     // of queries, of keys (and of values)
    int per_warp;  // all of them, or 1
    int warps;     // of a token
};

template <int D, bool HALF, bool ROPE>
__global__ void __launch_bounds__(QKV_THREADS, 8) k_paged_qkv(PagedQkvArgs a, Steps st) {
    pdl_enter();
    constexpr int LANES = D / 8, HEADS = 32 / LANES;  // lanes of a head, heads of a step
    constexpr int BATCH = 4;                          // steps whose reads are in flight together
    const int KV = a.cache.kv_heads, lane = threadIdx.x & 31, sub = lane % LANES, which = lane / LANES;
    const unsigned unit = blockIdx.x * (QKV_THREADS / 32) + (threadIdx.x >> 5);
    const unsigned token = unit / unsigned(st.warps);
    if (token >= unsigned(a.tokens)) return;  // a whole warp
    const int step0 = int(unit - token * st.warps) * st.per_warp, step1 = step0 + st.per_warp;
    const int slot = a.slots[token], position = ROPE ? a.positions[token] : 0;
    const bool live = slot >= 0 && slot < (long long)a.cache.pages * a.cache.page_size &&
                      (!ROPE || (position >= 0 && position < a.rope_rows));
    f32x2 cosine[2] = {0, 0}, sine[2] = {0, 0}, minus_sine[2] = {0, 0};
    if (ROPE) {
        const uint4 cs = __ldg(reinterpret_cast<const uint4*>(a.rope + (long long)(live ? position : 0) * (D / 2)) + sub);
        const uint32_t w[4] = {cs.x, cs.y, cs.z, cs.w};
#pragma unroll
        for (int e = 0; e < 2; e++) {
            cosine[e] = pair(lo_bf(w[2 * e]), lo_bf(w[2 * e + 1]));
            sine[e] = pair(hi_bf(w[2 * e]), hi_bf(w[2 * e + 1]));
            minus_sine[e] = pair(-hi_bf(w[2 * e]), -hi_bf(w[2 * e + 1]));
        }
    }
    const int page = live ? slot / a.cache.page_size : 0;
    const long long at = page * a.cache.page_stride + (slot - page * a.cache.page_size) * a.cache.token_stride + sub * 4;
    const uint16_t* const row = a.qkv + token * a.qkv_stride + sub * 4;

    // `count` heads from head `first` of the row on, whose first step is `base`: with a weight they are normed,
    // turned unless they are values, and go to dst, a head every `stride`.
    auto run = [&](int base, int first, int count, const uint16_t* norm, bool value, uint16_t* dst, long long stride, bool store) {
        f32x2 weight[4];
        if (norm) {
            const uint2 lo = __ldg(reinterpret_cast<const uint2*>(norm) + sub), hi = __ldg(reinterpret_cast<const uint2*>(norm + D / 2) + sub);
            weight[0] = widen<HALF>(lo.x);
            weight[1] = widen<HALF>(lo.y);
            weight[2] = widen<HALF>(hi.x);
            weight[3] = widen<HALF>(hi.y);
        }
        const int h0 = max(step0 - base, 0) * HEADS, h1 = min((step1 - base) * HEADS, count);
        for (int h = h0; h < h1; h += BATCH * HEADS) {
            uint2 v[BATCH][2];
            const uint16_t* src = row + (first + h + which) * D;
#pragma unroll
            for (int i = 0; i < BATCH; i++) {
                v[i][0] = v[i][1] = make_uint2(0u, 0u);
                if (h + i * HEADS + which < h1) {
                    v[i][0] = read_once(src + i * HEADS * D);
                    v[i][1] = read_once(src + i * HEADS * D + D / 2);
                }
            }
            uint16_t* to = dst + (h + which) * stride;
#pragma unroll
            for (int i = 0; i < BATCH; i++) {
                if (h + i * HEADS >= h1) break;  // the whole warp: all lanes reach the shuffles
                if (!value) {
                    f32x2 x[4] = {widen<HALF>(v[i][0].x), widen<HALF>(v[i][0].y), widen<HALF>(v[i][1].x), widen<HALF>(v[i][1].y)};
                    if (norm) {
                        f32x2 squares = mul2(x[0], x[0]);
#pragma unroll
                        for (int e = 1; e < 4; e++) squares = fma2(x[e], x[e], squares);
                        const float2 two = unpair(squares);
                        float ss = two.x + two.y;
#pragma unroll
                        for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(FULL_MASK, ss, o);
                        const float inv = rsqrtf(fmaf(ss, 1.0f / D, a.eps));
                        const f32x2 inv2 = pair(inv, inv);
#pragma unroll
                        for (int e = 0; e < 4; e++) x[e] = mul2(x[e], fma2(inv2, weight[e], inv2));  // x inv (1 + w)
                    }
                    if (ROPE) {  // without one, a turn by zero would mix 0 inf of the partner into a value
#pragma unroll
                        for (int half = 0; half < 2; half++) {
                            const f32x2 lo = x[half], hi = x[2 + half];
                            x[half] = fma2(lo, cosine[half], mul2(hi, minus_sine[half]));
                            x[2 + half] = fma2(hi, cosine[half], mul2(lo, sine[half]));
                        }
                    }
                    v[i][0] = make_uint2(narrow<HALF>(x[0]), narrow<HALF>(x[1]));
                    v[i][1] = make_uint2(narrow<HALF>(x[2]), narrow<HALF>(x[3]));
                }
                if (store && h + i * HEADS + which < h1) {
                    *reinterpret_cast<uint2*>(to + i * HEADS * stride) = live ? v[i][0] : make_uint2(0u, 0u);
                    *reinterpret_cast<uint2*>(to + i * HEADS * stride + D / 2) = live ? v[i][1] : make_uint2(0u, 0u);
                }
            }
        }
    };
    run(0, 0, a.heads, a.q_norm, false, a.q + token * a.q_stride + sub * 4, D, true);
    run(st.q, a.heads, KV, a.k_norm, false, a.cache.keys + at, a.cache.head_stride, live);
    run(st.q + st.kv, a.heads + KV, KV, nullptr, true, a.cache.values + at, a.cache.head_stride, live);
}

template <int D, bool HALF>
cudaError_t launch(const PagedQkvArgs& a, cudaStream_t s) {
    constexpr int WARPS = QKV_THREADS / 32, HEADS = 256 / D;
    Steps st;
    st.q = (a.heads + HEADS - 1) / HEADS;
    st.kv = (a.cache.kv_heads + HEADS - 1) / HEADS;
    const int steps = st.q + 2 * st.kv;
    // a step a warp while that leaves warps for no more than one round of 32 an SM
    st.per_warp = (long long)a.tokens * steps <= 148 * 32 ? 1 : steps;
    st.warps = steps / st.per_warp;
    const dim3 blocks(unsigned(((long long)a.tokens * st.warps + WARPS - 1) / WARPS));
    if (a.rope) return pdl_launch(k_paged_qkv<D, HALF, true>, blocks, dim3(QKV_THREADS), 0, s, a, st);
    return pdl_launch(k_paged_qkv<D, HALF, false>, blocks, dim3(QKV_THREADS), 0, s, a, st);
}

}  // namespace

cudaError_t launch_paged_qkv(const PagedQkvArgs& a, int head_dim, bool half, cudaStream_t s) {
    if (head_dim == 128) return half ? launch<128, true>(a, s) : launch<128, false>(a, s);
    return half ? launch<64, true>(a, s) : launch<64, false>(a, s);
}

}  // namespace plamo
