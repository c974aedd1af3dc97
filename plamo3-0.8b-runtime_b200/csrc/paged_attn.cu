// Attention of one new token of every request over its paged cache (plamo_k_paged_attention).
//
//   s_j = scale * q.k_j;  o = sum_j e^{s_j - m} v_j / sum_j e^{s_j - m};  lse = m + ln sum_j e^{s_j - m}
// in one pass over the keys with a running maximum and sum. Scores are kept in powers of two.
//
// A block takes one request and one KV head (at most 16 of its query heads: the rows of an m16n8k16 MMA;
// a larger group takes several blocks). Its four warps take every fourth 16-key tile, each with its own
// maximum, sum and output accumulators, and are joined in shared memory at the end. A tile's keys and
// values are copied with cp.async in an XOR-swizzled layout, so ldmatrix reads them without bank
// conflicts. Keys outside the visible range or without a page are filled with zeros and their scores
// replaced by -inf, so nothing stored there can reach a result.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "paged.h"

namespace plamo {
namespace {

constexpr int PA_THREADS = 128;
constexpr int PA_WARPS = PA_THREADS / 32;
constexpr int PA_HEADS = 16;  // query heads of a block: the MMA's rows
constexpr int PA_TILE = 16;   // keys of a tile

template <bool HALF>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (HALF)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool TRANS>
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    if (TRANS)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// 16 bytes into shared memory, or zeros where there is nothing to read.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}

// Probabilities enter the products as two 16-bit values, hi (cut off, not rounded) and lo = the rest +
// 2^-16 p: together p (1 + 2^-16) to 15 bits or more, a factor that P_PAIR takes out of the sum. Neither part
// of a p > 0 is zero or negative, so an infinite value times the pair is that infinity, never inf - inf or 0 inf.
constexpr float P_PAIR = 1.0f + 1.0f / 65536.0f;
template <bool HALF>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t& hi, uint32_t& lo) {
    constexpr float EXTRA = 1.0f / 65536.0f;
    if (HALF) {
        const __half2 h = __halves2half2(__float2half_rz(x), __float2half_rz(y));
        const float2 f = __half22float2(h);
        const __half2 l = __floats2half2_rn(fmaf(x, EXTRA, x - f.x), fmaf(y, EXTRA, y - f.y));
        hi = *reinterpret_cast<const uint32_t*>(&h);
        lo = *reinterpret_cast<const uint32_t*>(&l);
    } else {
        const uint32_t bx = __float_as_uint(x), by = __float_as_uint(y);
        hi = prmt(bx, by, 0x7632);
        const __nv_bfloat162 l = __floats2bfloat162_rn(fmaf(x, EXTRA, x - __uint_as_float(bx & 0xffff0000u)),
                                                       fmaf(y, EXTRA, y - __uint_as_float(by & 0xffff0000u)));
        lo = *reinterpret_cast<const uint32_t*>(&l);
    }
}
template <bool HALF>
__device__ __forceinline__ uint16_t round16(float x) {
    if (HALF) return __half_as_ushort(__float2half_rn(x));
    return __bfloat16_as_ushort(__float2bfloat16_rn(x));
}

// Running softmax of one warp: 16 heads (rows gq and gq + 8 of this lane) by D output columns.
template <int D>
struct Running {
    float m[2], l[2], o[D / 8][4];
    __device__ __forceinline__ void clear() {
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.f;
#pragma unroll
        for (int j = 0; j < D / 8; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) o[j][i] = 0.f;
    }
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// fp16 probabilities are held 2^14 times as large (at most 16384): the fp16 pair then keeps absolute
// errors below 2^-39 of the largest probability, where many tiny ones would otherwise be lost in
// subnormals. The sum carries the same factor, so only lse has to take it out. bf16 needs none.
template <bool HALF>
constexpr float P_SHIFT = HALF ? 14.f : 0.f;
// A maximum of -inf (nothing seen yet) is replaced by 0 where it is subtracted: e^{-inf - 0} = 0, not NaN.
__device__ __forceinline__ float origin(float m) { return m == -INFINITY ? 0.f : m; }

// Adds one tile of 16 keys (at kt, values at vt) of which those in `mask` are visible.
template <int D, bool HALF>
__device__ __forceinline__ void add_tile(Running<D>& run, const uint32_t (&qa)[D / 16][4], uint32_t kt, uint32_t vt,
                                         uint32_t mask, float scale) {
    const int lane = threadIdx.x & 31, tq = lane & 3;
    float acc[2][4];
#pragma unroll
    for (int n = 0; n < 2; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[n][i] = 0.f;
    // lanes 0-7 / 8-15 address keys 0-7 at the k-step's first / second chunk, 16-31 keys 8-15 likewise
    const int krow = (lane & 7) + ((lane >> 4) << 3), kchunk = (lane >> 3) & 1;
#pragma unroll
    for (int kk = 0; kk < D / 16; kk++) {
        uint32_t b[4];
        ldsm4<false>(b, kt + krow * (D * 2) + (((2 * kk + kchunk) ^ (krow & 7)) << 4));
        mma16816<HALF>(acc[0], qa[kk], b[0], b[1]);
        mma16816<HALF>(acc[1], qa[kk], b[2], b[3]);
    }
#pragma unroll
    for (int n = 0; n < 2; n++)
#pragma unroll
        for (int i = 0; i < 4; i++)
            acc[n][i] = (mask >> (8 * n + 2 * tq + (i & 1))) & 1u ? acc[n][i] * scale : -INFINITY;
    uint32_t ph[4], pl[4];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        float top = fmaxf(fmaxf(acc[0][2 * h], acc[0][2 * h + 1]), fmaxf(acc[1][2 * h], acc[1][2 * h + 1]));
        top = fmaxf(top, __shfl_xor_sync(FULL_MASK, top, 1));
        top = fmaxf(top, __shfl_xor_sync(FULL_MASK, top, 2));
        const float m = fmaxf(run.m[h], top), base = origin(m);
        const float fade = ex2(run.m[h] - base), origin_p = base - P_SHIFT<HALF>;
        run.m[h] = m;
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; i++) p[i] = ex2(acc[i >> 1][2 * h + (i & 1)] - origin_p);
        run.l[h] = fmaf(run.l[h], fade, (p[0] + p[1]) + (p[2] + p[3]));
        split_pair<HALF>(p[0], p[1], ph[h], pl[h]);
        split_pair<HALF>(p[2], p[3], ph[2 + h], pl[2 + h]);
#pragma unroll
        for (int j = 0; j < D / 8; j++) {
            run.o[j][2 * h] *= fade;
            run.o[j][2 * h + 1] *= fade;
        }
    }
    // lanes 0-15 address keys 0-15 of a chunk, lanes 16-31 those of the next
    const int vrow = lane & 15, vchunk = lane >> 4;
#pragma unroll
    for (int j = 0; j < D / 8; j += 2) {
        uint32_t b[4];
        ldsm4<true>(b, vt + vrow * (D * 2) + (((j + vchunk) ^ (vrow & 7)) << 4));
        mma16816<HALF>(run.o[j], ph, b[0], b[1]);
        mma16816<HALF>(run.o[j], pl, b[0], b[1]);
        mma16816<HALF>(run.o[j + 1], ph, b[2], b[3]);
        mma16816<HALF>(run.o[j + 1], pl, b[2], b[3]);
    }
}

template <int D, bool HALF>
__global__ void __launch_bounds__(PA_THREADS) k_paged_attn(PagedAttnArgs a, int group, int blocks_per_kv) {
    constexpr int ROW = D * 2, TILE_BYTES = PA_TILE * ROW, CH = D / 8;
    // the warps' tiles; afterwards the warps' outputs
    __shared__ __align__(128) uint8_t smem[PA_WARPS * PA_HEADS * D * 4];
    __shared__ float2 stats[PA_WARPS][PA_HEADS];
    static_assert(PA_WARPS * 2 * TILE_BYTES <= int(sizeof(smem)), "tiles fit");
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31, gq = lane >> 2, tq = lane & 3;
    const int r = blockIdx.y, kv = blockIdx.x / blocks_per_kv, h0 = (blockIdx.x % blocks_per_kv) * PA_HEADS;
    int qrow = r;
    if (a.row_start) {
        const int next = a.row_start[r + 1];
        if (next <= a.row_start[r]) return;
        qrow = next - 1;
    }
    if (qrow < 0 || qrow >= a.q_rows) return;
    const int heads = min(PA_HEADS, group - h0), head0 = kv * group + h0;
    const int n = min(max(a.lens[r], 0), a.max_len), first = a.window > 0 ? max(0, n - a.window) : 0;
    uint32_t qa[D / 16][4];
    const uint16_t* q = a.q + qrow * a.q_stride + head0 * D;
#pragma unroll
    for (int kk = 0; kk < D / 16; kk++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int h = gq + (i & 1) * 8, d = kk * 16 + 2 * tq + (i >> 1) * 8;
            qa[kk][i] = h < heads ? *reinterpret_cast<const uint32_t*>(q + h * D + d) : 0u;
        }
    Running<D> run;
    run.clear();
    const uint32_t kt = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * 2 * TILE_BYTES, vt = kt + TILE_BYTES;
    const int* table = a.table + size_t(r) * a.table_stride;
    for (int k0 = first + warp * PA_TILE; k0 < n; k0 += PA_WARPS * PA_TILE) {
        // lane j < 16 finds key j; the row's chunks are then copied by 16 (D = 128) or 8 lanes each
        long long at = -1;
        const int key = k0 + (lane & 15);
        if (key < n) {
            const int slot = key / a.cache.page_size, page = table[slot];
            if (page >= 0 && page < a.cache.pages)
                at = page * a.cache.page_stride + (key - slot * a.cache.page_size) * a.cache.token_stride +
                     kv * a.cache.head_stride;
        }
        const uint32_t mask = __ballot_sync(FULL_MASK, at >= 0) & 0xffffu;
#pragma unroll
        for (int i = 0; i < PA_TILE * CH / 32; i++) {
            const int row = i * (32 / CH) + lane / CH, c = lane % CH;
            const long long off = __shfl_sync(FULL_MASK, at, row);
            const uint32_t dst = row * ROW + ((c ^ (row & 7)) << 4);
            copy16(kt + dst, a.cache.keys + max(off, 0ll) + c * 8, off >= 0);
            copy16(vt + dst, a.cache.values + max(off, 0ll) + c * 8, off >= 0);
        }
        asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;" ::: "memory");
        __syncwarp();
        add_tile<D, HALF>(run, qa, kt, vt, mask, a.scale_log2);
        __syncwarp();
    }
    // join the warps
#pragma unroll
    for (int h = 0; h < 2; h++) {
        run.l[h] += __shfl_xor_sync(FULL_MASK, run.l[h], 1);
        run.l[h] += __shfl_xor_sync(FULL_MASK, run.l[h], 2);
        if (tq == 0) stats[warp][gq + 8 * h] = make_float2(run.m[h], run.l[h]);
    }
    __syncthreads();
    float* const part = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int j = 0; j < D / 8; j++)
#pragma unroll
        for (int h = 0; h < 2; h++)
            *reinterpret_cast<float2*>(part + (warp * PA_HEADS + gq + 8 * h) * D + j * 8 + 2 * tq) =
                make_float2(run.o[j][2 * h], run.o[j][2 * h + 1]);
    __syncthreads();
    for (int i = t; i < heads * D; i += PA_THREADS) {
        const int h = i / D;
        float m = -INFINITY;
        for (int w = 0; w < PA_WARPS; w++) m = fmaxf(m, stats[w][h].x);
        float l = 0.f, o = 0.f;
        for (int w = 0; w < PA_WARPS; w++) {
            const float f = ex2(stats[w][h].x - origin(m));
            l = fmaf(stats[w][h].y, f, l);
            o = fmaf(part[(w * PA_HEADS + h) * D + i % D], f, o);
        }
        a.out[qrow * a.out_stride + head0 * D + i] = round16<HALF>(o / (l > 0.f ? l * P_PAIR : 1.f));
        if (a.lse && i % D == 0)
            a.lse[size_t(qrow) * a.heads + head0 + h] = (origin(m) - P_SHIFT<HALF> + log2f(l)) * 0.693147180559945309f;
    }
}

}  // namespace

size_t paged_attention_workspace() { return 1 << 20; }

cudaError_t launch_paged_attention(const PagedAttnArgs& a, int head_dim, bool half, cudaStream_t s) {
    const int group = a.heads / a.cache.kv_heads, per_kv = (group + PA_HEADS - 1) / PA_HEADS;
    const dim3 grid(a.cache.kv_heads * per_kv, a.rows);
    if (head_dim == 128) {
        if (half) k_paged_attn<128, true><<<grid, PA_THREADS, 0, s>>>(a, group, per_kv);
        else k_paged_attn<128, false><<<grid, PA_THREADS, 0, s>>>(a, group, per_kv);
    } else {
        if (half) k_paged_attn<64, true><<<grid, PA_THREADS, 0, s>>>(a, group, per_kv);
        else k_paged_attn<64, false><<<grid, PA_THREADS, 0, s>>>(a, group, per_kv);
    }
    return cudaGetLastError();
}

}  // namespace plamo
