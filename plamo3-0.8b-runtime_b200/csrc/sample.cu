// Sampling by temperature, top-k, top-p and min-p from given uniform numbers (plamo_k_sample).
//
//   w_i = floor(2^40 exp((x_i - max x) / T)) as whole numbers, so sums are exact in any order;
//   kept: a run of the order (x descending, index ascending): the first k, of those the shortest run with
//   at least p of their weight, of those the ones with w >= min_p 2^40;
//   id = the lowest kept index whose running weight (in index order) exceeds floor(2^24 u) W / 2^24.
// The kept run is described by a threshold on the order-preserving key of x and by how many of the values
// at the threshold belong to it, so nothing is sorted.
//
// A cluster of up to 8 blocks takes a row: each keeps its slice of the logits in shared memory after one
// read from global memory, and sums and histograms are exchanged through distributed shared memory, one
// cluster barrier each. A threshold takes a histogram over 1024 equal steps of (max - x), which spreads
// the many near-equal logits that bins by bits of x would pile onto a few addresses, then one over the
// keys inside the chosen step (one for 16-bit logits, mostly two for fp32). What cannot be kept is skipped
// before its exponential is taken: w = 0 beyond 27.8 T, and under top-p what V times over would not fill the
// part that may be left out. Bound by instructions (an exponential an id at least) for many rows, by the
// cluster barriers (3 to 9) for one.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"
#include "paged.h"

namespace plamo {
namespace {

namespace cg = cooperative_groups;

constexpr int SAMPLE_THREADS = 512;
constexpr int SAMPLE_WARPS = SAMPLE_THREADS / 32;
constexpr int BINS = 1024;
constexpr int MAX_CLUSTER = 8;
constexpr int SLICE_BYTES = 128 * 1024;  // most of a slice kept in shared memory; the rest is read again
constexpr float SPAN = 27.8f;            // 2^40 exp(-27.8) < 1
typedef unsigned long long u64;

template <int TYPE>
struct Logit;
template <>
struct Logit<0> {  // bf16
    typedef uint16_t raw;
    static constexpr int KEY_SHIFT = 16;  // bits of the fp32 key that are the same for every value
    static constexpr uint16_t NOTHING = 0xff80;
    static __device__ __forceinline__ float value(uint16_t b) { return bf2f(b); }
};
template <>
struct Logit<1> {  // fp16
    typedef uint16_t raw;
    static constexpr int KEY_SHIFT = 13;
    static constexpr uint16_t NOTHING = 0xfc00;
    static __device__ __forceinline__ float value(uint16_t b) { return __half2float(__ushort_as_half(b)); }
};
template <>
struct Logit<2> {  // fp32
    typedef uint32_t raw;
    static constexpr int KEY_SHIFT = 0;
    static constexpr uint32_t NOTHING = 0xff800000u;
    static __device__ __forceinline__ float value(uint32_t b) { return __uint_as_float(b); }
};

// Order-preserving key of a logit (larger is larger, -0 equals 0).
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
template <int SHIFT>
__device__ __forceinline__ float key_value(uint32_t k) {
    const uint32_t full = k << SHIFT;
    if (full & 0x80000000u) return __uint_as_float(full & 0x7fffffffu);
    return __uint_as_float(~(full | ((1u << SHIFT) - 1u)));
}

// x > -inf
__device__ __forceinline__ u64 weight(float x, float top, float temperature) {
    const float e = x == top ? 1.f : expf(__fdiv_rn(x - top, temperature));
    return e > 0.f ? u64(e * 1099511627776.0f) : 0ull;
}

// fraction * total / 2^24 in whole numbers (fraction <= 2^24, total < 2^62), rounded down or up
__device__ __forceinline__ u64 share(u64 fraction, u64 total, bool up) {
    return fraction * (total >> 24) + ((fraction * (total & 0xffffffull) + (up ? 0xffffffull : 0ull)) >> 24);
}

__device__ __forceinline__ u64 warp_add(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL_MASK, v, o);
    return v;
}

struct Pair {
    u64 a, b;
};

struct Shared {
    u64 hist[2][BINS];  // two, used in turn: one may still be read by other blocks while the next fills
    Pair exchange[4];   // likewise
    Pair warp_pairs[SAMPLE_WARPS];
    u64 scan[SAMPLE_WARPS];
    // a histogram's answer: the bin, the amount before it, the amount in it
    u64 bin, before, amount;
};

template <int TYPE>
struct Row {
    typedef typename Logit<TYPE>::raw raw;
    static constexpr int VEC = 16 / sizeof(raw);
    cg::cluster_group cluster = cg::this_cluster();
    Shared& sh;
    raw* slice;           // the block's slice, `cached` values of it
    const raw* row;
    int vocab, rank, ranks;
    int lead;             // the row begins `lead` values after a 16-byte boundary: value j is id j - lead
    int begin, length, cached;  // the block's values [begin, begin + length)
    int mine0, mine1;     // this thread's values, from begin
    int turn = 0, hist_turn = 0;
    float top, temperature;

    __device__ Row(Shared& s) : sh(s) {}

    __device__ __forceinline__ raw raw_at(int i) const {
        if (i < cached) return slice[i];
        const int id = begin + i - lead;
        return id >= 0 && id < vocab ? row[id] : Logit<TYPE>::NOTHING;
    }
    __device__ __forceinline__ float at(int i) const { return Logit<TYPE>::value(raw_at(i)); }
    static __device__ __forceinline__ uint32_t key(float x) { return order_key(x) >> Logit<TYPE>::KEY_SHIFT; }

    // Sums of both values over the block.
    __device__ __forceinline__ Pair block_add(Pair v) {
        v.a = warp_add(v.a);
        v.b = warp_add(v.b);
        __syncthreads();
        if ((threadIdx.x & 31) == 0) sh.warp_pairs[threadIdx.x >> 5] = v;
        __syncthreads();
        Pair s = threadIdx.x % 32 < SAMPLE_WARPS ? sh.warp_pairs[threadIdx.x % 32] : Pair{0, 0};
        s.a = warp_add(s.a);
        s.b = warp_add(s.b);
        return s;
    }
    // Every block's pair (already summed over the block) becomes known to all: their sum, and the sum over the
    // blocks before this one.
    __device__ __forceinline__ Pair exchange(Pair block, Pair& before) {
        Pair* const place = &sh.exchange[turn++ & 3];
        if (threadIdx.x == 0) *place = block;
        cluster.sync();
        const int lane = threadIdx.x & 31;
        Pair p{0, 0};
        if (lane < ranks) p = *cluster.map_shared_rank(place, lane);
        before.a = warp_add(lane < rank ? p.a : 0ull);
        before.b = warp_add(lane < rank ? p.b : 0ull);
        return Pair{warp_add(p.a), warp_add(p.b)};
    }
    // Exclusive running sum over the block in thread order.
    __device__ __forceinline__ u64 block_scan(u64 v) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        u64 x = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 y = __shfl_up_sync(FULL_MASK, x, o);
            if (lane >= o) x += y;
        }
        __syncthreads();
        if (lane == 31) sh.scan[warp] = x;
        __syncthreads();
        u64 before = 0;
#pragma unroll
        for (int w = 0; w < SAMPLE_WARPS; w++) before += w < warp ? sh.scan[w] : 0ull;
        return before + x - v;
    }

    // One histogram over the cluster. classify(x) gives a value's bin (larger values in lower bins) or -1; an
    // entry counts 1, or its weight. Finds the first bin at which `base` and the amounts up to it reach `need`
    // (left in sh.bin / before / amount); false when they do not.
    template <bool WEIGHTS, typename F>
    __device__ __forceinline__ bool histogram(F classify, u64 base, u64 need) {
        u64* const hist = sh.hist[hist_turn++ & 1];
        uint32_t* const counts = reinterpret_cast<uint32_t*>(hist);
        for (int i = threadIdx.x; i < BINS; i += SAMPLE_THREADS) {
            if (WEIGHTS) hist[i] = 0;
            else counts[i] = 0;
        }
        if (threadIdx.x == 0) sh.bin = BINS;
        __syncthreads();
        for (int i = mine0; i < mine1; i++) {
            const float x = at(i);
            const int bin = classify(x);
            if (bin < 0) continue;
            if (WEIGHTS) {
                const u64 w = weight(x, top, temperature);
                if (w) atomicAdd(hist + bin, w);
            } else {
                atomicAdd(counts + bin, 1u);
            }
        }
        cluster.sync();
        constexpr int PER = BINS / SAMPLE_THREADS;
        u64 sum[PER], all = 0;
#pragma unroll
        for (int b = 0; b < PER; b++) sum[b] = 0;
        for (int c = 0; c < ranks; c++) {
            const u64* const h = cluster.map_shared_rank(hist, c);
            const uint32_t* const n = reinterpret_cast<const uint32_t*>(h);
#pragma unroll
            for (int b = 0; b < PER; b++) sum[b] += WEIGHTS ? h[threadIdx.x * PER + b] : n[threadIdx.x * PER + b];
        }
#pragma unroll
        for (int b = 0; b < PER; b++) all += sum[b];
        u64 before = base + block_scan(all);
#pragma unroll
        for (int b = 0; b < PER; b++) {
            if (before < need && need <= before + sum[b]) {
                sh.bin = threadIdx.x * PER + b;
                sh.before = before;
                sh.amount = sum[b];
            }
            before += sum[b];
        }
        __syncthreads();
        return sh.bin < BINS;
    }

    // The key at which the amounts of the values, from the largest down, reach `need`; before and amount: the
    // amounts above it and at it. Values more than `limit` below the largest do not matter. False when the
    // amounts stay below `need`.
    template <bool WEIGHTS>
    __device__ __forceinline__ bool find(u64 need, float limit, uint32_t least_key, uint32_t& edge, u64& before, u64& amount) {
        const float step = float(BINS) / limit;
        auto coarse = [&](float x) -> int {
            const float d = top - x;
            if (!(x > -INFINITY) || d > limit) return -1;
            return min(int(d * step), BINS - 1);
        };
        auto within = [&](float x) -> int { return key(x) < least_key ? -1 : coarse(x); };
        if (!histogram<WEIGHTS>(within, 0, need)) return false;
        const int bin = int(sh.bin);
        u64 base = sh.before;
        // keys that the bin can hold: its bounds, widened by more than the two roundings of `coarse`
        const double low = bin == BINS - 1 ? double(limit) : (bin + 1) / double(step), high = bin ? bin / double(step) : 0.0;
        uint32_t khi = key(__double2float_ru(double(top) - high * (1.0 - 1e-6)));
        uint32_t klo = key(__double2float_rd(double(top) - low * (1.0 + 1e-6)));
        if (top == INFINITY) khi = klo = key(top);
        while (true) {
            const int bits = 32 - __clz(khi - klo), shift = max(bits - 10, 0);
            __syncthreads();  // the answer before has been read
            auto fine = [&](float x) -> int {
                const uint32_t k = key(x);
                return k < least_key || k > khi || k < klo || coarse(x) != bin ? -1 : int((khi - k) >> shift);
            };
            if (!histogram<WEIGHTS>(fine, base, need)) return false;  // cannot happen: the bin holds it
            base = sh.before;
            khi -= uint32_t(sh.bin) << shift;
            if (!shift) break;
            klo = max(klo, khi - ((1u << shift) - 1u));
        }
        edge = khi;
        before = base;
        amount = sh.amount;
        __syncthreads();
        return true;
    }
};

template <int TYPE>
__global__ void __launch_bounds__(SAMPLE_THREADS) k_sample(SampleArgs a, int slice_len, int cached) {
    pdl_enter();
    typedef typename Logit<TYPE>::raw raw;
    extern __shared__ __align__(16) uint8_t sample_smem[];
    __shared__ Shared shared;
    Row<TYPE> row(shared);
    constexpr int VEC = Row<TYPE>::VEC;
    const int t = threadIdx.x, V = a.vocab;
    row.ranks = int(row.cluster.num_blocks());
    row.rank = int(row.cluster.block_rank());
    const int r = blockIdx.x / row.ranks;
    row.row = static_cast<const raw*>(a.logits) + r * a.row_stride;
    row.slice = reinterpret_cast<raw*>(sample_smem);
    row.vocab = V;
    row.lead = int((reinterpret_cast<uintptr_t>(row.row) & 15) / sizeof(raw));
    row.begin = row.rank * slice_len;
    row.length = min(max(V + row.lead - row.begin, 0), slice_len);
    row.cached = min(cached, row.length);
    // an odd number of values a thread: neighbouring threads start in different banks
    const int per = ((row.length + SAMPLE_THREADS - 1) / SAMPLE_THREADS) | 1;
    row.mine0 = min(t * per, row.length);
    row.mine1 = min(row.mine0 + per, row.length);

    float T = a.temperature ? a.temperature[r] : 1.f;
    const bool warm = T > 0.f;
    if (!warm) T = 1.f;
    int k = !warm ? 1 : a.top_k ? a.top_k[r] : 0;
    if (k <= 0 || k > V) k = V;
    const float top_p = a.top_p ? a.top_p[r] : 1.f, min_p = a.min_p ? a.min_p[r] : 0.f, u = a.u[r];
    const u64 p24 = top_p < 1.f ? u64(rint(fmax(double(top_p), 0.0) * 16777216.0)) : 1ull << 24;
    const u64 least = max(1ull, min_p > 0.f ? u64(ceil(fmin(double(min_p), 1.0) * 1099511627776.0)) : 0ull);
    row.temperature = T;

    // read the slice once; the largest logit (fmaxf passes over NaN)
    float top = -INFINITY;
    for (int v = t; v * VEC < row.length; v += SAMPLE_THREADS) {
        const int j = v * VEC, id = row.begin + j - row.lead;
        raw x[VEC];
        if (id >= 0 && id + VEC <= V) {
            *reinterpret_cast<uint4*>(x) = __ldg(reinterpret_cast<const uint4*>(row.row + id));
        } else {
#pragma unroll
            for (int e = 0; e < VEC; e++) x[e] = id + e >= 0 && id + e < V ? row.row[id + e] : Logit<TYPE>::NOTHING;
        }
        if (j < row.cached) *reinterpret_cast<uint4*>(row.slice + j) = *reinterpret_cast<const uint4*>(x);
#pragma unroll
        for (int e = 0; e < VEC; e++) top = fmaxf(top, Logit<TYPE>::value(x[e]));
    }
    top = warp_max(top);
    Pair unused;
    {
        Pair* const place = &shared.exchange[row.turn++ & 3];
        if ((t & 31) == 0) shared.scan[t >> 5] = __float_as_uint(top);
        __syncthreads();
        top = warp_max(t % 32 < SAMPLE_WARPS ? __uint_as_float(uint32_t(shared.scan[t % 32])) : -INFINITY);
        if (t == 0) place->a = __float_as_uint(top);
        row.cluster.sync();
        const int lane = t & 31;
        top = warp_max(lane < row.ranks ? __uint_as_float(uint32_t(row.cluster.map_shared_rank(place, lane)->a)) : -INFINITY);
    }
    row.top = top;

    // kept: keys above `edge`, and the first `ties` (in index order) of the `at_edge` values at it
    uint32_t edge = 0;
    u64 ties = 0, at_edge = 0, before, amount;
    if (k < V && row.template find<false>(k, SPAN * T, 0u, edge, before, amount)) {
        at_edge = amount;
        ties = k - before;
    }
    if (p24 < (1ull << 24)) {
        Pair w{0, 0};
        const float far = SPAN * T;
        for (int i = row.mine0; i < row.mine1; i++) {
            const float x = row.at(i);
            if (x > -INFINITY && !(top - x > far) && row.key(x) >= edge) w.a += weight(x, top, T);
        }
        const u64 one = ties < at_edge ? weight(key_value<Logit<TYPE>::KEY_SHIFT>(edge), top, T) : 0ull;
        const u64 run = row.exchange(row.block_add(w), unused).a - (at_edge - ties) * one;
        const u64 need = max(share(p24, run, true), 1ull);
        // an id whose weight V times over fits into what may be left out is left out itself
        const u64 small = (run - min(need, run)) / u64(V);
        const float limit = small > 1 ? fminf(far, T * (log2f(1099511627776.0f / float(small)) * 0.6931472f) * 1.0001f + 1e-6f * T) : far;
        uint32_t cut = edge;
        if (run && row.template find<true>(need, limit, edge, cut, before, amount)) {
            const u64 each = weight(key_value<Logit<TYPE>::KEY_SHIFT>(cut), top, T);
            ties = (need - before + each - 1) / each;
            at_edge = amount / each;
            edge = cut;
        }
    }
    // ranks of the values at the edge, where only some of them are kept
    u64 first_tie = 0;
    if (ties < at_edge) {
        u64 n = 0;
        for (int i = row.mine0; i < row.mine1; i++) {
            const float x = row.at(i);
            n += x > -INFINITY && row.key(x) == edge;
        }
        Pair ahead;
        row.exchange(row.block_add({n, 0}), ahead);
        first_tie = ahead.a + row.block_scan(n);
    }
    const float far = SPAN * T;
    auto kept_weight = [&](int i, u64& tie) -> u64 {
        const float x = row.at(i);
        if (!(x > -INFINITY) || top - x > far) return 0ull;
        const uint32_t key = row.key(x);
        if (key < edge || (key == edge && ties < at_edge && tie++ >= ties)) return 0ull;
        const u64 w = weight(x, top, T);
        return w >= least ? w : 0ull;
    };
    Pair mine{0, 0};
    u64 tie = first_tie;
    for (int i = row.mine0; i < row.mine1; i++) {
        const u64 w = kept_weight(i, tie);
        mine.a += w;
        mine.b += w != 0;
    }
    Pair ahead;
    const Pair total = row.exchange(row.block_add(mine), ahead);
    const u64 m = u > 0.f ? min(u64(fminf(u, 1.f) * 16777216.0f), (1ull << 24) - 1) : 0ull;
    const u64 target = share(m, total.a, false);
    u64 upto = ahead.a + row.block_scan(mine.a);
    if (upto <= target && target < upto + mine.a) {
        tie = first_tie;
        for (int i = row.mine0; i < row.mine1; i++) {
            const u64 w = kept_weight(i, tie);
            if (target < upto + w) {
                a.ids[r] = row.begin + i - row.lead;
                if (a.logprobs) a.logprobs[r] = float(log(double(w) / double(total.a)));
                break;
            }
            upto += w;
        }
    }
    if (row.rank == 0 && t == 0) {
        if (a.kept) a.kept[r] = int(total.b);
        if (!total.a) {
            a.ids[r] = 0;
            if (a.logprobs) a.logprobs[r] = -INFINITY;
        }
    }
    row.cluster.sync();  // no block leaves while another may read its shared memory
}

template <int TYPE>
cudaError_t launch(const SampleArgs& a, cudaStream_t s) {
    constexpr int SIZE = TYPE == 2 ? 4 : 2, VEC = 16 / SIZE;
    // blocks a row: enough to keep slices in shared memory, more while the rows leave SMs idle
    int ranks = 1;
    while (ranks < MAX_CLUSTER && ((long long)a.vocab * SIZE > (long long)ranks * SLICE_BYTES / 2 || a.rows * ranks < 296) &&
           a.vocab / ranks > 2048)
        ranks *= 2;
    const int len = ((a.vocab + VEC - 1 + ranks - 1) / ranks + VEC - 1) / VEC * VEC;
    const int cached = std::min(len, SLICE_BYTES / SIZE);
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_shared(k_sample<TYPE>, SLICE_BYTES, done);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(a.rows) * ranks);
    cfg.blockDim = dim3(SAMPLE_THREADS);
    cfg.dynamicSmemBytes = size_t(cached) * SIZE;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, k_sample<TYPE>, a, len, cached);
}

}  // namespace

cudaError_t launch_sample(const SampleArgs& a, int dtype, cudaStream_t s) {
    return dtype == 0 ? launch<0>(a, s) : dtype == 1 ? launch<1>(a, s) : launch<2>(a, s);
}

}  // namespace plamo
