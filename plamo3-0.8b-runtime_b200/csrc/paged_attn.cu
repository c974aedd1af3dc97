// Attention of one new token of every request over its paged cache (plamo_k_paged_attention).
//
//   s_j = scale * q.k_j;  o = sum_j e^{s_j - m} v_j / sum_j e^{s_j - m};  lse = m + ln sum_j e^{s_j - m}
// in one pass over the keys with a running maximum and sum. Scores are kept in powers of two.
//
// Split. The work is a line of units (64 keys of one request and one KV head, at most 16 of its query
// heads: the rows of an m16n8k16 MMA), request after request, with a few empty places before each request
// and head for what beginning it costs. Each block takes one stretch of equal length of that line,
// whatever the lengths are, so a batch of any raggedness ends in one wave. The lengths are
// on the device: every block adds them up itself. A request and head inside one stretch is finished there;
// one that is cut leaves an fp32 partial per block, and k_paged_join adds those up in order, so a
// result does not depend on timing. Calls whose requests cannot be cut launch no join.
//
// Block. Four warps take every fourth 16-key tile of a stretch, each with its own running maximum, sum and
// outputs and its own ring of tiles: no barrier inside the loop. A tile's keys and values are copied with
// cp.async in an XOR-swizzled layout, so ldmatrix reads them without bank conflicts; the page lookup of a
// tile runs one tile ahead of its copy. Tiles begin at positions that are multiples of 16, so where the
// page size is one too a tile lies in one page and has one lookup; else each key has its own. Keys
// outside the visible range or without a page are filled with zeros and their scores replaced by -inf, so
// nothing stored there can reach a result.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "paged.h"

#include <algorithm>
#include <climits>
#include <type_traits>

namespace plamo {
namespace {

namespace cg = cooperative_groups;

constexpr int PA_THREADS = 128;
constexpr int PA_WARPS = PA_THREADS / 32;
constexpr int PA_HEADS = 16;  // query heads of a block: the MMA's rows
constexpr int PA_TILE = 16;   // keys of a tile
constexpr int PA_UNIT = 64;   // keys of a unit: one tile for each warp
// Requests of at most this many keys are one unit and never cut.
constexpr int PA_WHOLE = 256;
// What beginning a request and head costs a block, in units: its share of the line is that much longer.
constexpr int PA_BEGIN = 3;
// A cluster of up to 8 blocks takes a request and head, of the largest size that all of them run at once at, where a
// block's share of the longest request is at most this many keys: the first number always, the second when the
// blocks fill most SMs. Cluster and line, us: 64 x 512 keys 7.2 and 10.7, 148 x 500 12.4 and 16.9, 32 x 2048 11.0
// and 13.7, 48 x 2048 14.5 and 16.5. Past the second number even lengths still gain (40 x 3000 to 4000: 18.4 and
// 20.5) but ragged ones lose, as the longest request holds up its cluster alone (74 x 100 to 2000: 14.8 and 12.7;
// 18 x 100 to 2000, 4 KV heads: 13.7 and 11.3). The host knows max_len alone, not the lengths: under a bound far above
// them a call takes the line (1 x 700 keys: 7.2 us under 32768, 5.9 under 700; 64 x 512: 10.6 and 7.2).
constexpr int PA_CLUSTER = 8;
constexpr int PA_SHARE = 264;
constexpr int PA_SHARE_FULL = 640;
constexpr int PA_MAX_BLOCKS = 592;
// tiles in a warp's ring: 96 KB a block, two blocks an SM
template <int D>
constexpr int PA_STAGES = 384 / D;

template <bool HALF>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (HALF)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
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
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// 16 bytes into shared memory, or zeros where there is nothing to read.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}

// Probabilities enter the products as two 16-bit values, hi (cut off, not rounded) and lo = the rest +
// 2^-16 p: together p (1 + 2^-16) to 15 bits or more, a factor that P_PAIR takes out of the sum. Neither part of a
// p > 0 is negative, and neither may vanish, so an infinite value times the pair is that infinity, never inf - inf
// or 0 inf: a part that has rounded to zero is raised to the least the type holds (fp16: 2^-24, by P_SHIFT 2^-38 of the
// largest probability; bf16: 2^-126, its least normal number). p itself is zero below 2^-126 of the largest.
// Two parts move 0.3 to 0.7% of the bf16 outputs by one step of the type against a softmax that keeps all 24 bits, and
// leave their error against 64 bits the same to four digits: the outputs' own rounding is far larger. A third part
// would bring that to 0.05% (64 x 32768 keys: 0.4%), for 4% (1 x 700) to 8% (48 requests, window 2048) more time.
constexpr float P_PAIR = 1.0f + 1.0f / 65536.0f;
template <bool HALF>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t& hi, uint32_t& lo) {
    constexpr float EXTRA = 1.0f / 65536.0f;
    const uint32_t bx = __float_as_uint(x), by = __float_as_uint(y), cut = prmt(bx, by, 0x7632);
    // positive 16-bit floats order as whole numbers do; the upper half of an fp32 p is zero for p = 0 alone
    const uint32_t least = __vminu2(cut, HALF ? 0x00010001u : 0x00800080u);
    if (HALF) {
        const __half2 h = __halves2half2(__float2half_rz(x), __float2half_rz(y));
        const float2 f = __half22float2(h);
        const __half2 l = __floats2half2_rn(fmaf(x, EXTRA, x - f.x), fmaf(y, EXTRA, y - f.y));
        hi = __vmaxu2(*reinterpret_cast<const uint32_t*>(&h), least);
        lo = __vmaxu2(*reinterpret_cast<const uint32_t*>(&l), least);
    } else {
        hi = cut;
        const __nv_bfloat162 l = __floats2bfloat162_rn(fmaf(x, EXTRA, x - __uint_as_float(bx & 0xffff0000u)),
                                                       fmaf(y, EXTRA, y - __uint_as_float(by & 0xffff0000u)));
        lo = __vmaxu2(*reinterpret_cast<const uint32_t*>(&l), least);
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

// 2^x to 2^-22 of itself; results below 2^-126 are zero, which no sum beside a largest probability of 1 can show.
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

// Where a lane's ldmatrix and copy addresses lie in a tile, the same for every tile: the swizzle repeats every 8
// chunks and every 8 rows, so four offsets and constants beside them are enough.
template <int D>
struct Offsets {
    static constexpr int ROW = D * 2, CH = D / 8, RPS = 32 / CH, COPIES = 8 / RPS;  // rows a step of copies, steps of 8 rows
    uint32_t key[4], value[4], copy[COPIES];
    __device__ __forceinline__ Offsets() {
        const int lane = threadIdx.x & 31;
        // keys: lanes 0-7 / 8-15 address keys 0-7 at a k-step's first / second chunk, 16-31 keys 8-15 likewise
        const int krow = (lane & 7) + ((lane >> 4) << 3), kchunk = (lane >> 3) & 1;
        // values: lanes 0-15 address keys 0-15 of a chunk, lanes 16-31 those of the next
        const int vrow = lane & 15, vchunk = lane >> 4;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            key[i] = krow * ROW + (((2 * i + kchunk) ^ (krow & 7)) << 4);
            value[i] = vrow * ROW + (((2 * i + vchunk) ^ (vrow & 7)) << 4);
        }
#pragma unroll
        for (int i = 0; i < COPIES; i++) {
            const int row = i * RPS + lane / CH;
            copy[i] = row * ROW + (((lane % CH) ^ (row & 7)) << 4);
        }
    }
};

// Adds one tile of 16 keys (at kt, values behind them) of which those in `mask` are visible. upper: there are more
// than 8 heads (rows 8 to 15 of the MMA); without it their softmax is skipped.
template <int D, bool HALF>
__device__ __forceinline__ void add_tile(Running<D>& run, const uint32_t (&qa)[D / 16][4], const Offsets<D>& off, uint32_t kt,
                                         uint32_t mask, float scale, bool upper) {
    const int tq = threadIdx.x & 3;
    // even and odd k-steps are added up apart: half the length of a chain of dependent MMAs
    float acc[2][4], odd[2][4];
#pragma unroll
    for (int n = 0; n < 2; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[n][i] = odd[n][i] = 0.f;
#pragma unroll
    for (int kk = 0; kk < D / 16; kk++) {
        uint32_t b[4];
        ldsm4<false>(b, kt + off.key[kk & 3] + (kk >> 2) * 128);
        mma16816<HALF>(kk & 1 ? odd[0] : acc[0], qa[kk], b[0], b[1]);
        mma16816<HALF>(kk & 1 ? odd[1] : acc[1], qa[kk], b[2], b[3]);
    }
#pragma unroll
    for (int n = 0; n < 2; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[n][i] += odd[n][i];
    if (mask != 0xffffu) {
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (!((mask >> (8 * n + 2 * tq + (i & 1))) & 1u)) acc[n][i] = -INFINITY;
    }
    uint32_t ph[4], pl[4];
    float fade[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        if (h == 1 && !upper) {
            fade[1] = 1.f;
            ph[1] = ph[3] = pl[1] = pl[3] = 0u;
            break;
        }
        float top = fmaxf(fmaxf(acc[0][2 * h], acc[0][2 * h + 1]), fmaxf(acc[1][2 * h], acc[1][2 * h + 1]));
        top = fmaxf(top, __shfl_xor_sync(FULL_MASK, top, 1));
        top = fmaxf(top, __shfl_xor_sync(FULL_MASK, top, 2));
        // the scale is positive: it does not change which score is the largest
        const float m = fmaxf(run.m[h], top * scale), base = origin(m), origin_p = base - P_SHIFT<HALF>;
        fade[h] = ex2(run.m[h] - base);
        run.m[h] = m;
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; i++) p[i] = ex2(fmaf(acc[i >> 1][2 * h + (i & 1)], scale, -origin_p));
        run.l[h] = fmaf(run.l[h], fade[h], (p[0] + p[1]) + (p[2] + p[3]));
        split_pair<HALF>(p[0], p[1], ph[h], pl[h]);
        split_pair<HALF>(p[2], p[3], ph[2 + h], pl[2 + h]);
    }
    // most tiles leave every maximum where it was
    if (__any_sync(FULL_MASK, fade[0] != 1.f || fade[1] != 1.f)) {
#pragma unroll
        for (int j = 0; j < D / 8; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) run.o[j][i] *= fade[i >> 1];
    }
    const uint32_t vt = kt + PA_TILE * D * 2;
#pragma unroll
    for (int j = 0; j < D / 8; j += 4) {
        uint32_t b[2][4];
#pragma unroll
        for (int g = 0; g < 2; g++) ldsm4<true>(b[g], vt + off.value[(j / 2 + g) & 3] + (j >> 3) * 128);
        // the two products of an output are four MMAs apart
#pragma unroll
        for (int g = 0; g < 4; g++) mma16816<HALF>(run.o[j + g], ph, b[g >> 1][2 * (g & 1)], b[g >> 1][2 * (g & 1) + 1]);
#pragma unroll
        for (int g = 0; g < 4; g++) mma16816<HALF>(run.o[j + g], pl, b[g >> 1][2 * (g & 1)], b[g >> 1][2 * (g & 1) + 1]);
    }
}

// Four finished outputs of a head, and its lse.
template <bool HALF>
__device__ __forceinline__ void store_row(const PagedAttnArgs& a, int qrow, int head, int D, int d, float4 o, float m, float l) {
    if (l == 0.f) o = make_float4(0.f, 0.f, 0.f, 0.f);  // no score above -inf: zeros, whatever the values made of 0 p
    const float inv = 1.0f / (l > 0.f ? l * P_PAIR : 1.f);
    uint2 w;
    w.x = round16<HALF>(o.x * inv) | uint32_t(round16<HALF>(o.y * inv)) << 16;
    w.y = round16<HALF>(o.z * inv) | uint32_t(round16<HALF>(o.w * inv)) << 16;
    *reinterpret_cast<uint2*>(a.out + qrow * a.out_stride + head * D + d) = w;
    if (a.lse && d == 0) a.lse[size_t(qrow) * a.heads + head] = (origin(m) - P_SHIFT<HALF> + log2f(l)) * 0.693147180559945309f;
}

int sm_count() {
    static const int n = [] {
        int dev = 0, v = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) v = 148;
        return std::min(v, PA_MAX_BLOCKS / 2);
    }();
    return n;
}

// What k_paged_join needs of one request and head: its query row (-1: nothing to join), heads, and the pieces, of
// which blocks first_block ... first_block + pieces - 1 hold one each.
struct __align__(16) JoinRecord {
    int qrow, head0, heads, pieces;
    int first_slot, first_block, unused0, unused1;
};
// Workspace: 2 partials a block (of the first and the last request of its stretch), each 16 heads x head_dim
// outputs, then 2 x 16 (maximum, sum) pairs a block, then the join's records.
constexpr size_t PA_STATS_AT = size_t(2) * PA_MAX_BLOCKS * PA_HEADS * 128 * sizeof(float);
constexpr size_t PA_RECORDS_AT = PA_STATS_AT + size_t(2) * PA_MAX_BLOCKS * PA_HEADS * sizeof(float2);
constexpr size_t PA_WORKSPACE = PA_RECORDS_AT + size_t(PA_MAX_BLOCKS) * sizeof(JoinRecord);

struct Split {
    int unit;       // keys of a unit
    int pairs;      // (KV head, block of 16 query heads) pairs of a request
    int per_kv;     // blocks of 16 query heads of a KV head
    int group;      // query heads of a KV head
    int page_shift; // log2 of the page size, -1 when it is no power of two
    int blocks;     // of k_paged_attn
    int join;       // 0: no request can be cut; 1: records by (request, pair); 2: by block of k_paged_attn
};

// The query row of request r, -1 when it has none.
__device__ __forceinline__ int query_row(const PagedAttnArgs& a, int r) {
    int q = r;
    if (a.row_start) {
        q = a.row_start[r + 1] - 1;
        if (q < a.row_start[r]) return -1;
    }
    return q >= 0 && q < a.q_rows ? q : -1;
}

// The line of work: upto[r] places lie before request r.
struct Line {
    const int* upto;
    int total, per_block;
    // A request and head, and where on the line they are.
    struct Place {
        int r, pair, begin, length;
    };
    __device__ __forceinline__ int begin_of(int block) const { return int(min((long long)block * per_block, (long long)total)); }
    __device__ __forceinline__ Place at(int x, int rows, int pairs) const {
        // the last request that begins at or before x
        int lo = 0, hi = rows - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (upto[mid] * pairs <= x) lo = mid;
            else hi = mid - 1;
        }
        Place p;
        p.r = lo;
        p.length = upto[lo + 1] - upto[lo];
        const int inside = x - upto[lo] * pairs;
        p.pair = pairs == 1 ? 0 : inside / p.length;
        p.begin = x - (inside - p.pair * p.length);
        return p;
    }
};

// What a request of length n sees: keys [first, end). Units and tiles begin at `origin`, first rounded down to a tile.
struct Seen {
    int first, end, origin;
    __device__ __forceinline__ Seen(const PagedAttnArgs& a, int n) {
        end = min(max(n, 0), a.max_len);
        first = a.window > 0 ? max(0, end - a.window) : 0;
        origin = first & ~(PA_TILE - 1);
    }
};

// Every block adds up the requests' places itself: the lengths are on the device, and this costs one read of
// them. `upto` is shared memory for rows + 1 sums.
template <int THREADS>
__device__ __forceinline__ Line lay_out(const PagedAttnArgs& a, const Split& sp, int* upto) {
    __shared__ int warp_sums[THREADS / 32];
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const int per = (a.rows + THREADS - 1) / THREADS, r0 = min(t * per, a.rows), r1 = min(r0 + per, a.rows);
    int sum = 0;
    for (int r = r0; r < r1; r++) {
        const Seen seen(a, a.lens[r]);
        const int units = query_row(a, r) >= 0 ? (seen.end - seen.origin + sp.unit - 1) / sp.unit : 0;
        const int places = units ? units + PA_BEGIN : 0;
        upto[r + 1] = places;
        sum += places;
    }
    int x = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(FULL_MASK, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    int at = x - sum;
    for (int w = 0; w < warp; w++) at += warp_sums[w];
    for (int r = r0; r < r1; r++) {
        at += upto[r + 1];
        upto[r + 1] = at;
    }
    if (t == 0) upto[0] = 0;
    __syncthreads();
    Line line;
    line.upto = upto;
    line.total = upto[a.rows] * sp.pairs;  // below 2^31 by the choice of the unit
    line.per_block = max(1, int((unsigned(line.total) + sp.blocks - 1u) / unsigned(sp.blocks)));
    return line;
}

// A block's work on one request and KV head: keys [k0, k1) (k0 at a tile's beginning, nothing before `first` is
// visible), of whose tiles warp number `warp` of `warps` takes every warps-th.
struct Work {
    int r, kv, head0, heads, qrow, first, k0, k1, warp, warps;
};
template <int D>
constexpr int PA_PITCH = D + 8;  // a warp's outputs, a head a row: 8 floats further than a multiple of 32 banks

// Runs the warp's tiles, and leaves the warps' outputs (relative to the block's maximum, PA_PITCH floats a head) in
// the rings' place and their (maximum, sum) pairs in `stats`. Ends with a barrier.
template <int D, bool HALF, bool ALIGNED>
__device__ __forceinline__ void attend(const PagedAttnArgs& a, const Split& sp, const Work& w, uint8_t* smem,
                                       float2 (*stats)[PA_HEADS]) {
    constexpr int ROW = D * 2, TILE_BYTES = PA_TILE * ROW, CH = D / 8, S = PA_STAGES<D>, PITCH = PA_PITCH<D>;
    static_assert(PA_HEADS * PITCH * 4 <= S * 2 * TILE_BYTES, "a warp's outputs fit in its ring");
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31, gq = lane >> 2, tq = lane & 3;
    const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * S * 2 * TILE_BYTES;
    const Offsets<D> at;
    constexpr int RPS = Offsets<D>::RPS, COPIES = Offsets<D>::COPIES;
    const int c = lane % CH, row0 = lane / CH;  // this lane copies chunk c of rows row0, row0 + RPS, ...
    const int* table = a.table + size_t(w.r) * a.table_stride;
    const int tiles = (w.k1 - w.k0 + PA_TILE - 1) / PA_TILE;
    const int mine = tiles > w.warp ? (tiles - w.warp + w.warps - 1) / w.warps : 0;  // tiles w.warp, w.warp + w.warps, ...
    const uint16_t* const keys = a.cache.keys + w.kv * a.cache.head_stride + c * 8;
    const uint16_t* const values = a.cache.values + w.kv * a.cache.head_stride + c * 8;
    const long long step = RPS * a.cache.token_stride;
    auto page_index = [&](int key) { return sp.page_shift >= 0 ? key >> sp.page_shift : key / a.cache.page_size; };
    // The page of the tile at key0 (ALIGNED), or of its key `lane % 16`; -1 outside the range.
    auto page_of = [&](int key0) -> int {
        const int key = key0 + (ALIGNED ? 0 : lane & 15);
        return key < w.k1 ? __ldg(table + page_index(key)) : -1;
    };
    // Copies the tile at key0 to kt, values behind its keys; which of its keys are visible.
    auto issue = [&](int key0, int page, uint32_t kt) -> uint32_t {
        uint32_t mask = 0xffffu;
        if (key0 < w.first || key0 + PA_TILE > w.k1)
            mask = ((1u << min(w.k1 - key0, PA_TILE)) - 1u) & ~((1u << max(w.first - key0, 0)) - 1u);
        const bool held = page >= 0 && page < a.cache.pages;
        long long off = 0;  // of this lane's first row (ALIGNED), or of key `lane % 16`
        if (ALIGNED) {
            if (!held) mask = 0u;
            off = page * a.cache.page_stride + (key0 - page_index(key0) * a.cache.page_size + row0) * a.cache.token_stride;
        } else {
            const int key = key0 + (lane & 15);
            if (held) off = page * a.cache.page_stride + (key - page_index(key) * a.cache.page_size) * a.cache.token_stride;
            mask &= __ballot_sync(FULL_MASK, held) & 0xffffu;
        }
        if (mask == 0xffffu) {
#pragma unroll
            for (int i = 0; i < PA_TILE / RPS; i++) {
                const uint32_t dst = kt + at.copy[i % COPIES] + (i / COPIES) * 8 * ROW;
                const long long from = ALIGNED ? off : __shfl_sync(FULL_MASK, off, i * RPS + row0);
                copy16(dst, keys + from);
                copy16(dst + TILE_BYTES, values + from);
                if (ALIGNED) off += step;
            }
        } else {
#pragma unroll 1
            for (int i = 0; i < PA_TILE / RPS; i++) {
                const int row = i * RPS + row0;
                const uint32_t dst = kt + row * ROW + ((c ^ (row & 7)) << 4);
                const long long from = ALIGNED ? off : __shfl_sync(FULL_MASK, off, row);
                const bool valid = mask >> row & 1u;
                copy16(dst, valid ? keys + from : a.cache.keys, valid);
                copy16(dst + TILE_BYTES, valid ? values + from : a.cache.values, valid);
                if (ALIGNED) off += step;
            }
        }
        return mask;
    };
    const int stride = w.warps * PA_TILE;
    int key0 = w.k0 + w.warp * PA_TILE, ahead = key0;  // the next tile to copy, and to look up
    int pages[S];  // the lookups of the next tiles to copy, the ring's first ones together
#pragma unroll
    for (int i = 0; i < S; i++, ahead += stride) pages[i] = page_of(ahead);
    // the queries wait in the ring's last place until it is needed
    const uint32_t qt = ring + (S - 1) * 2 * TILE_BYTES;
    const uint16_t* const q = a.q + w.qrow * a.q_stride + w.head0 * D + c * 8;
    if (mine)
#pragma unroll
        for (int i = 0; i < PA_TILE / RPS; i++) {
            const int row = i * RPS + row0;
            copy16(qt + at.copy[i % COPIES] + (i / COPIES) * 8 * ROW, row < w.heads ? q + row * D : a.q, row < w.heads);
        }
    asm volatile("cp.async.commit_group;" ::: "memory");
    uint32_t qa[D / 16][4];
    Running<D> run;
    run.clear();
    // tile j is copied while tile j - (S - 1) is worked on
    uint32_t masks[S], to = ring, from = ring;
    const uint32_t ring_end = ring + S * 2 * TILE_BYTES;
#pragma unroll
    for (int i = 0; i < S; i++) masks[i] = 0u;
#pragma unroll 1
    for (int j = 0; j < mine + S - 1; j++) {
        if (j == S - 1) {
            asm volatile("cp.async.wait_group %0;" ::"n"(S - 1) : "memory");
            __syncwarp();
            // the heads are addressed as the values' keys are
#pragma unroll
            for (int kk = 0; kk < D / 16; kk++) ldsm4<false>(qa[kk], qt + at.value[kk & 3] + (kk >> 2) * 128);
            __syncwarp();
        }
        masks[S - 1] = j < mine ? issue(key0, pages[0], to) : 0u;
        asm volatile("cp.async.commit_group;" ::: "memory");
        key0 += stride;
        to = to + 2 * TILE_BYTES == ring_end ? ring : to + 2 * TILE_BYTES;
#pragma unroll
        for (int i = 0; i < S - 1; i++) pages[i] = pages[i + 1];
        pages[S - 1] = page_of(ahead);
        ahead += stride;
        if (j >= S - 1) {
            asm volatile("cp.async.wait_group %0;" ::"n"(S - 1) : "memory");
            __syncwarp();
            add_tile<D, HALF>(run, qa, at, from, masks[0], a.scale_log2, w.heads > 8);
            __syncwarp();  // the tile has been read: the next copy may overwrite it
            from = from + 2 * TILE_BYTES == ring_end ? ring : from + 2 * TILE_BYTES;
        }
#pragma unroll
        for (int i = 0; i < S - 1; i++) masks[i] = masks[i + 1];
    }
    // join the warps
#pragma unroll
    for (int h = 0; h < 2; h++) {
        run.l[h] += __shfl_xor_sync(FULL_MASK, run.l[h], 1);
        run.l[h] += __shfl_xor_sync(FULL_MASK, run.l[h], 2);
        if (tq == 0) stats[warp][gq + 8 * h] = make_float2(run.m[h], run.l[h]);
    }
    __syncthreads();  // every warp is done with its ring
    float* const mid = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int h = 0; h < 2; h++) {
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < PA_WARPS; w++) m = fmaxf(m, stats[w][gq + 8 * h].x);
        const float f = ex2(run.m[h] - origin(m));
#pragma unroll
        for (int j = 0; j < D / 8; j++)
            *reinterpret_cast<float2*>(mid + (warp * PA_HEADS + gq + 8 * h) * PITCH + j * 8 + 2 * tq) =
                make_float2(run.o[j][2 * h] * f, run.o[j][2 * h + 1] * f);
    }
    __syncthreads();
}

// Four outputs of one head, added up over the block's warps: item counts heads, and D / 4 pieces of a head.
template <int D>
__device__ __forceinline__ float4 block_sum(const uint8_t* smem, const float2 (*stats)[PA_HEADS], int h, int d, float& m, float& l) {
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int w = 0; w < PA_WARPS; w++) m = fmaxf(m, stats[w][h].x);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < PA_WARPS; w++) {
        const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem) + (w * PA_HEADS + h) * PA_PITCH<D> + d);
        l = fmaf(stats[w][h].y, ex2(stats[w][h].x - origin(m)), l);
        o.x += v.x;
        o.y += v.y;
        o.z += v.z;
        o.w += v.w;
    }
    return o;
}

// A query row that sees nothing: zeros, and -inf.
__device__ __forceinline__ void store_nothing(const PagedAttnArgs& a, int qrow, int head0, int heads, int D) {
    for (int i = threadIdx.x; i < heads * D; i += blockDim.x) a.out[qrow * a.out_stride + head0 * D + i] = 0;
    if (a.lse)
        for (int h = threadIdx.x; h < heads; h += blockDim.x) a.lse[size_t(qrow) * a.heads + head0 + h] = -INFINITY;
}

constexpr size_t ring_bytes(int D) { return size_t(PA_WARPS) * (384 / D) * 2 * PA_TILE * D * 2; }

// The line's kernel. The sums of more than about 4000 requests no longer leave an SM room for two blocks (requests of 200
// to 900 keys: 4000 in 191 us, 4200 in 306).
template <int D, bool HALF, bool ALIGNED>
__global__ void __launch_bounds__(PA_THREADS, 2) k_paged_attn(PagedAttnArgs a, Split sp) {
    pdl_enter();
    extern __shared__ __align__(128) uint8_t pa_smem[];
    // the warps' rings, then the running sums of the requests' places
    int* const upto = reinterpret_cast<int*>(pa_smem + ring_bytes(D));  // [rows + 1]
    __shared__ float2 stats[PA_WARPS][PA_HEADS];
    const int t = threadIdx.x;
    float* const parts = static_cast<float*>(a.workspace);
    float2* const part_stats = reinterpret_cast<float2*>(static_cast<uint8_t*>(a.workspace) + PA_STATS_AT);
    const Line line = lay_out<PA_THREADS>(a, sp, upto);
    const int x0 = line.begin_of(blockIdx.x), x1 = line.begin_of(blockIdx.x + 1);

    JoinRecord* const records = reinterpret_cast<JoinRecord*>(static_cast<uint8_t*>(a.workspace) + PA_RECORDS_AT);
    for (int r = blockIdx.x; r < a.rows; r += gridDim.x) {
        if (upto[r + 1] != upto[r]) continue;
        if (sp.join == 1)
            for (int p = t; p < sp.pairs; p += PA_THREADS) records[r * sp.pairs + p].qrow = -1;
        const int qrow = query_row(a, r);
        if (qrow >= 0) store_nothing(a, qrow, 0, a.heads, D);
    }
    if (sp.join == 2 && x0 >= x1 && t == 0) records[blockIdx.x].qrow = -1;

    for (int x = x0; x < x1;) {
        const Line::Place at = line.at(x, a.rows, sp.pairs);
        const int units = at.length - PA_BEGIN, place = x - at.begin;
        const int stop = min(at.length, place + (x1 - x));
        const int u = max(place - PA_BEGIN, 0), take = stop - PA_BEGIN - u;  // its units here: [u, u + take)
        const int slot = 2 * blockIdx.x + (x != x0);
        Work w;
        w.r = at.r;
        w.kv = sp.per_kv == 1 ? at.pair : at.pair / sp.per_kv;
        const int h0 = (at.pair - w.kv * sp.per_kv) * PA_HEADS;
        w.heads = min(PA_HEADS, sp.group - h0);
        w.head0 = w.kv * sp.group + h0;
        w.qrow = query_row(a, at.r);
        if (sp.join && t == 0) {
            const int b0 = (at.begin + PA_BEGIN) / line.per_block, b1 = (at.begin + at.length - 1) / line.per_block;
            const JoinRecord rec{b1 > b0 ? w.qrow : -1, w.head0, w.heads, b1 - b0 + 1, 2 * b0 + (at.begin > b0 * line.per_block), b0, 0, 0};
            if (sp.join == 1) {
                if (u == 0 && take > 0) records[at.r * sp.pairs + at.pair] = rec;
            } else if (x == x0) {  // a cut request's record stands with its second block
                records[blockIdx.x] = rec;
                if (int(blockIdx.x) != b0 + 1) records[blockIdx.x].qrow = -1;
            }
        }
        x += stop - place;
        if (take <= 0) continue;
        const Seen seen(a, a.lens[at.r]);
        w.first = seen.first;
        w.k0 = seen.origin + u * sp.unit;
        w.k1 = int(min((long long)seen.end, w.k0 + (long long)take * sp.unit));
        w.warp = t >> 5;
        w.warps = PA_WARPS;
        attend<D, HALF, ALIGNED>(a, sp, w, pa_smem, stats);
#pragma unroll
        for (int i = 0; i < PA_HEADS * D / 4 / PA_THREADS; i++) {
            const int item = i * PA_THREADS + t, h = item / (D / 4), d = (item % (D / 4)) * 4;
            if (h >= w.heads) break;
            float m, l;
            const float4 o = block_sum<D>(pa_smem, stats, h, d, m, l);
            if (take == units) {
                store_row<HALF>(a, w.qrow, w.head0 + h, D, d, o, m, l);
            } else {
                *reinterpret_cast<float4*>(parts + (size_t(slot) * PA_HEADS + h) * D + d) = o;
                if (d == 0) part_stats[slot * PA_HEADS + h] = make_float2(m, l);
            }
        }
        __syncthreads();  // the rings and stats are free again
    }
}

// The kernel of few requests of moderate length: a cluster takes one request and head, its warps every tile in
// turn, and the blocks' sums are joined through distributed shared memory, each block taking some heads. One
// launch, no line to lay out and no join.
template <int D, bool HALF, bool ALIGNED>
__global__ void __launch_bounds__(PA_THREADS, 2) k_paged_attn_cluster(PagedAttnArgs a, Split sp) {
    pdl_enter();
    extern __shared__ __align__(128) uint8_t pa_smem[];
    __shared__ float2 stats[PA_WARPS][PA_HEADS];
    __shared__ float2 sums[PA_HEADS];
    // the block's outputs, behind the warps'
    constexpr int AT = PA_WARPS * PA_HEADS * PA_PITCH<D> * 4;
    static_assert(AT + PA_HEADS * D * 4 <= int(ring_bytes(D)), "the block's outputs fit behind the warps'");
    float* const part = reinterpret_cast<float*>(pa_smem + AT);
    cg::cluster_group cluster = cg::this_cluster();
    const int t = threadIdx.x, ranks = int(cluster.num_blocks()), rank = int(cluster.block_rank());
    const int at = blockIdx.x / ranks;  // the request and head
    Work w;
    w.r = at / sp.pairs;
    const int pair = at - w.r * sp.pairs;
    w.kv = sp.per_kv == 1 ? pair : pair / sp.per_kv;
    const int h0 = (pair - w.kv * sp.per_kv) * PA_HEADS;
    w.heads = min(PA_HEADS, sp.group - h0);
    w.head0 = w.kv * sp.group + h0;
    w.qrow = query_row(a, w.r);
    if (w.qrow < 0) return;  // the whole cluster
    const Seen seen(a, a.lens[w.r]);
    if (seen.end <= seen.first) {
        if (rank == 0) store_nothing(a, w.qrow, w.head0, w.heads, D);
        return;
    }
    w.first = seen.first;
    w.k0 = seen.origin;
    w.k1 = seen.end;
    w.warp = rank * PA_WARPS + (t >> 5);
    w.warps = ranks * PA_WARPS;
    attend<D, HALF, ALIGNED>(a, sp, w, pa_smem, stats);
#pragma unroll
    for (int i = 0; i < PA_HEADS * D / 4 / PA_THREADS; i++) {
        const int item = i * PA_THREADS + t, h = item / (D / 4), d = (item % (D / 4)) * 4;
        float m, l;
        *reinterpret_cast<float4*>(part + h * D + d) = block_sum<D>(pa_smem, stats, h, d, m, l);
        if (d == 0) sums[h] = make_float2(m, l);
    }
    cluster.sync();
    const int share = (PA_HEADS + ranks - 1) / ranks;  // heads of a block
    for (int item = t; item < share * (D / 4); item += PA_THREADS) {
        const int h = rank * share + item / (D / 4), d = (item % (D / 4)) * 4;
        if (h >= w.heads) break;
        float2 st[PA_CLUSTER];
        float4 v[PA_CLUSTER];
#pragma unroll
        for (int c = 0; c < PA_CLUSTER; c++) {  // all reads in flight together
            st[c] = make_float2(-INFINITY, 0.f);
            v[c] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (c < ranks) {
                st[c] = cluster.map_shared_rank(sums, c)[h];
                v[c] = *reinterpret_cast<const float4*>(cluster.map_shared_rank(part, c) + h * D + d);
            }
        }
        float m = -INFINITY, l = 0.f;
#pragma unroll
        for (int c = 0; c < PA_CLUSTER; c++) m = fmaxf(m, st[c].x);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int c = 0; c < PA_CLUSTER; c++) {
            const float f = ex2(st[c].x - origin(m));
            l = fmaf(st[c].y, f, l);
            o.x = fmaf(v[c].x, f, o.x);
            o.y = fmaf(v[c].y, f, o.y);
            o.z = fmaf(v[c].z, f, o.z);
            o.w = fmaf(v[c].w, f, o.w);
        }
        store_row<HALF>(a, w.qrow, w.head0 + h, D, d, o, m, l);
    }
    cluster.sync();  // no block leaves while another reads its sums
}

// Adds BATCH pieces, every PER_HEAD-th from p0 on, of head h to a lane's (m, l, o), all reads in flight together.
// Past the last piece the last is read again and left out: reads under a condition were waited for one after
// another (32 requests of 0 to 2048 keys: 14.8 us the call, so 10.8).
template <int D, int PER_HEAD, int BATCH>
__device__ __forceinline__ void add_pieces(const JoinRecord& rec, const float* parts, const float2* part_stats, int p0, int h,
                                           float& m, float& l, float (&o)[D / 32]) {
    constexpr int VEC = D / 32;
    typedef typename std::conditional<D == 128, float4, float2>::type Vec;
    const int lane = threadIdx.x & 31;
    float2 st[BATCH];
    __align__(16) float v[BATCH][VEC];
#pragma unroll
    for (int b = 0; b < BATCH; b++) {
        const int p = min(p0 + b * PER_HEAD, rec.pieces - 1), slot = p == 0 ? rec.first_slot : 2 * (rec.first_block + p);
        st[b] = part_stats[slot * PA_HEADS + h];
        *reinterpret_cast<Vec*>(v[b]) = *reinterpret_cast<const Vec*>(parts + (size_t(slot) * PA_HEADS + h) * D + lane * VEC);
    }
#pragma unroll
    for (int b = 0; b < BATCH; b++) {
        if (p0 + b * PER_HEAD < rec.pieces) continue;
        st[b] = make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int i = 0; i < VEC; i++) v[b][i] = 0.f;
    }
#pragma unroll
    for (int b = 0; b < BATCH; b++) {
        const float top = fmaxf(m, st[b].x), fade = ex2(m - origin(top)), f = ex2(st[b].x - origin(top));
        l = fmaf(st[b].y, f, l * fade);
#pragma unroll
        for (int i = 0; i < VEC; i++) o[i] = fmaf(v[b][i], f, o[i] * fade);
        m = top;
    }
}

// Adds up the pieces of the heads of a cut request, block x those of record x. A block takes WARPS / PER_HEAD heads,
// PER_HEAD warps each: a warp adds every PER_HEAD-th piece, 8 reads in flight together, then the warps of a head are
// added. What to add stands in the records that k_paged_attn left: the lengths are not read again.
template <int D, bool HALF, int WARPS, int PER_HEAD>
__global__ void __launch_bounds__(WARPS * 32) k_paged_join(PagedAttnArgs a) {
    pdl_enter();
    constexpr int VEC = D / 32;
    typedef typename std::conditional<D == 128, float4, float2>::type Vec;
    __shared__ __align__(16) float outs[WARPS][D];
    __shared__ float2 stats[WARPS];
    const JoinRecord rec =
        reinterpret_cast<const JoinRecord*>(static_cast<const uint8_t*>(a.workspace) + PA_RECORDS_AT)[blockIdx.x];
    if (rec.qrow < 0) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int h = blockIdx.y * (WARPS / PER_HEAD) + warp / PER_HEAD, part = warp % PER_HEAD;
    const float* const parts = static_cast<const float*>(a.workspace);
    const float2* const part_stats = reinterpret_cast<const float2*>(static_cast<const uint8_t*>(a.workspace) + PA_STATS_AT);
    float m = -INFINITY, l = 0.f;
    __align__(16) float o[VEC];
#pragma unroll
    for (int i = 0; i < VEC; i++) o[i] = 0.f;
    const bool inside = h < rec.heads;
    for (int p0 = inside ? part : rec.pieces; p0 < rec.pieces;) {
        if (rec.pieces - p0 > 4 * PER_HEAD) {
            add_pieces<D, PER_HEAD, 8>(rec, parts, part_stats, p0, h, m, l, o);
            p0 += 8 * PER_HEAD;
        } else {
            add_pieces<D, PER_HEAD, 4>(rec, parts, part_stats, p0, h, m, l, o);
            p0 += 4 * PER_HEAD;
        }
    }
    *reinterpret_cast<Vec*>(&outs[warp][lane * VEC]) = *reinterpret_cast<const Vec*>(o);
    if (lane == 0) stats[warp] = make_float2(m, l);
    if (PER_HEAD == 1) __syncwarp();
    else __syncthreads();
    if (part != 0 || !inside || lane * 4 >= D) return;
    const int d = lane * 4;
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int i = 0; i < PER_HEAD; i++) top = fmaxf(top, stats[warp + i].x);
    float4 out = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < PER_HEAD; i++) {
        const float f = ex2(stats[warp + i].x - origin(top));
        const float4 v = *reinterpret_cast<const float4*>(&outs[warp + i][d]);
        sum = fmaf(stats[warp + i].y, f, sum);
        out.x = fmaf(v.x, f, out.x);
        out.y = fmaf(v.y, f, out.y);
        out.z = fmaf(v.z, f, out.z);
        out.w = fmaf(v.w, f, out.w);
    }
    store_row<HALF>(a, rec.qrow, rec.head0 + h, D, d, out, top, sum);
}

template <int D, bool HALF, bool ALIGNED>
cudaError_t launch_main(const PagedAttnArgs& a, const Split& sp, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_shared(k_paged_attn<D, HALF, ALIGNED>, ring_bytes(D) + (PAGED_MAX_ROWS + 1) * sizeof(int), done);
    if (e != cudaSuccess) return e;
    return pdl_launch(k_paged_attn<D, HALF, ALIGNED>, dim3(sp.blocks), dim3(PA_THREADS), ring_bytes(D) + (a.rows + 1) * sizeof(int), s,
                      a, sp);
}

template <int D, bool HALF, bool ALIGNED>
struct Cluster {
    static void configure(cudaLaunchConfig_t& cfg, cudaLaunchAttribute (&attr)[2], unsigned clusters, int ranks, cudaStream_t s) {
        cfg = {};
        cfg.gridDim = dim3(clusters * ranks);
        cfg.blockDim = dim3(PA_THREADS);
        cfg.dynamicSmemBytes = ring_bytes(D);
        cfg.stream = s;
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = ranks;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
        cfg.attrs = attr;
        cfg.numAttrs = 2;
    }
    // How many clusters of `ranks` blocks run at once (asked once; a cluster stays within a group of SMs, so this
    // is less than the blocks would allow: 33 of 8, 45 of 6, 56 of 5, 71 of 4, 93 of 3 on 148 SMs).
    static int fit(int ranks) {
        static std::atomic<int> known[PA_CLUSTER + 1];
        int n = known[ranks].load();
        if (n) return n;
        static std::atomic<uint64_t> done{0};
        if (allow_shared(k_paged_attn_cluster<D, HALF, ALIGNED>, ring_bytes(D), done) != cudaSuccess) return 0;
        cudaLaunchConfig_t cfg;
        cudaLaunchAttribute attr[2];
        configure(cfg, attr, 1, ranks, nullptr);
        cfg.numAttrs = 1;
        if (cudaOccupancyMaxActiveClusters(&n, k_paged_attn_cluster<D, HALF, ALIGNED>, &cfg) != cudaSuccess) n = 0;
        known[ranks].store(n);
        return n;
    }
    static cudaError_t launch(const PagedAttnArgs& a, const Split& sp, int ranks, cudaStream_t s) {
        static std::atomic<uint64_t> done{0};
        cudaError_t e = allow_shared(k_paged_attn_cluster<D, HALF, ALIGNED>, ring_bytes(D), done);
        if (e != cudaSuccess) return e;
        cudaLaunchConfig_t cfg;
        cudaLaunchAttribute attr[2];
        configure(cfg, attr, unsigned(a.rows) * sp.pairs, ranks, s);
        return cudaLaunchKernelEx(&cfg, k_paged_attn_cluster<D, HALF, ALIGNED>, a, sp);
    }
    // The largest cluster that runs all requests and heads at once, 0 where the line is faster.
    static int ranks(long long pairs, long long longest) {
        for (int r = PA_CLUSTER; r > 1; r--)
            if (pairs <= fit(r)) return longest <= r * (pairs * r >= 0.8 * sm_count() ? PA_SHARE_FULL : PA_SHARE) ? r : 0;
        return 0;
    }
};

template <int D, bool HALF>
cudaError_t launch(const PagedAttnArgs& a, cudaStream_t s) {
    Split sp;
    sp.group = a.heads / a.cache.kv_heads;
    sp.per_kv = (sp.group + PA_HEADS - 1) / PA_HEADS;
    sp.pairs = a.cache.kv_heads * sp.per_kv;
    sp.page_shift = -1;
    for (int i = 0; i < 31; i++)
        if (a.cache.page_size == 1 << i) sp.page_shift = i;
    // keys from the first tile on
    const long long longest = a.window > 0 ? std::min((long long)a.window + PA_TILE - 1, (long long)a.max_len) : a.max_len;
    const bool aligned = a.cache.page_size % PA_TILE == 0;
    if (longest > PA_WHOLE) {
        const long long pairs = (long long)a.rows * sp.pairs;
        const int ranks = aligned ? Cluster<D, HALF, true>::ranks(pairs, longest) : Cluster<D, HALF, false>::ranks(pairs, longest);
        if (ranks)
            return aligned ? Cluster<D, HALF, true>::launch(a, sp, ranks, s) : Cluster<D, HALF, false>::launch(a, sp, ranks, s);
    }
    // short requests stay whole; units grow only where their number would pass 31 bits
    long long unit = longest <= PA_WHOLE ? PA_WHOLE : PA_UNIT;
    while (a.rows * ((longest + unit - 1) / unit + PA_BEGIN) * sp.pairs > INT_MAX / 2) unit *= 2;
    sp.unit = int(unit);
    const long long units = (longest + unit - 1) / unit;
    sp.blocks = int(std::min(a.rows * sp.pairs * (units > 1 ? units + PA_BEGIN : 1), 2ll * sm_count()));
    const int pairs = a.rows * sp.pairs;
    sp.join = units <= 1 ? 0 : pairs <= sp.blocks ? 1 : 2;
    cudaError_t e = aligned ? launch_main<D, HALF, true>(a, sp, s) : launch_main<D, HALF, false>(a, sp, s);
    if (e != cudaSuccess || !sp.join) return e;
    // More warps a head where a head has more pieces (about blocks / pairs). The call in us with 16, 8, 4 and 1 warps a
    // head: 6 x 20000 keys, 49 pieces: 18.6, 19.3; 12 x 9000, 25 pieces: 18.1, 16.3, 17.0, 19.0; 40 x 100 to 4000, 7
    // pieces: 15.2, 11.8, 11.0, 12.6; 74 x 100 to 2000, 4 pieces: 19.7, 13.9, 13.1, 12.5.
    const int records = sp.join == 1 ? pairs : sp.blocks, heads = std::min(sp.group, PA_HEADS);
    if (sp.blocks > 40 * pairs) return pdl_launch(k_paged_join<D, HALF, 16, 16>, dim3(records, heads), dim3(512), 0, s, a);
    if (sp.blocks > 15 * pairs) return pdl_launch(k_paged_join<D, HALF, 8, 8>, dim3(records, heads), dim3(256), 0, s, a);
    if (sp.blocks > 5 * pairs) return pdl_launch(k_paged_join<D, HALF, 8, 4>, dim3(records, (heads + 1) / 2), dim3(256), 0, s, a);
    return pdl_launch(k_paged_join<D, HALF, 4, 1>, dim3(records, (heads + 3) / 4), dim3(128), 0, s, a);
}

}  // namespace

size_t paged_attention_workspace() { return PA_WORKSPACE; }

cudaError_t launch_paged_attention(const PagedAttnArgs& a, int head_dim, bool half, cudaStream_t s) {
    if (head_dim == 128) return half ? launch<128, true>(a, s) : launch<128, false>(a, s);
    return half ? launch<64, true>(a, s) : launch<64, false>(a, s);
}

}  // namespace plamo
