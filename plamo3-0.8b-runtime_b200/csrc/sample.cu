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
// cluster barrier each. What is kept is nearly always a small head of the vocabulary, so the aim is to name a
// superset of it of at most 1024 ids, which the first block sorts and finishes alone:
// - under top-k, the values from the j-th largest of 128 thread groups' maxima up: for k up to half the groups j = k,
//   as k values are at least that large; for k up to twice the groups the j that leaves a quarter more than k if large
//   values lie anywhere (n ids spread over N groups miss N e^{-n/N} of them), and k are counted. Else, and when
//   that fails, those up to the step of a histogram where k is reached;
// - under top-p, the values within 8.3 T of the top (there, one in 4000 as likely), beside the sum of all weights.
//   When those do not hold p or are too many, a histogram of what could be kept at all (what V times over would fit
//   into the part left out cannot) gives the step where p is reached. Histograms have 256 equal steps of
//   (max - x), which spreads the many near-equal logits that bins by bits of x would pile onto a few addresses.
// A larger superset has its threshold narrowed down by histograms over the keys inside the step, and all
// blocks finish the row. w = 0 beyond 27.8 T. Bound by the instructions of the passes over the ids (an exponential
// an id at least, unless top-k comes first) and their latencies for many rows: 64 x 80,001 fp32 unfiltered use half of the
// issue slots at 7 warps a scheduler, 32 x 107,520 of mixed controls a third at 4. By the cluster barriers for one.
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
constexpr int BINS = 256;
constexpr int LIST = 1024;               // ids that the first block can finish alone
constexpr int FEW = 128;                 // ids that are compared each with each rather than sorted
constexpr int MAX_CLUSTER = 8;
constexpr int GROUPS = MAX_CLUSTER * SAMPLE_WARPS;  // of a cluster: a warp of 8 blocks, ... 4 lanes of one
// Most of a slice kept in shared memory; the rest is read again by every pass, value by value (8 rows of 262,144 fp32
// ids, which fit: 12.1 us unfiltered; of 400,001: 38.7).
constexpr int SLICE_BYTES = 128 * 1024;
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
    // the larger of two pairs of values (or of one), and the larger value of a pair; NaN loses
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
        const __nv_bfloat162 m = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
        return *reinterpret_cast<const uint32_t*>(&m);
    }
    static __device__ __forceinline__ float larger(uint32_t a) { return fmaxf(lo_bf(a), hi_bf(a)); }
    static constexpr uint32_t NOTHING2 = 0xff80ff80u;
};
template <>
struct Logit<1> {  // fp16
    typedef uint16_t raw;
    static constexpr int KEY_SHIFT = 13;
    static constexpr uint16_t NOTHING = 0xfc00;
    static __device__ __forceinline__ float value(uint16_t b) { return __half2float(__ushort_as_half(b)); }
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
        const __half2 m = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
        return *reinterpret_cast<const uint32_t*>(&m);
    }
    static __device__ __forceinline__ float larger(uint32_t a) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&a));
        return fmaxf(f.x, f.y);
    }
    static constexpr uint32_t NOTHING2 = 0xfc00fc00u;
};
template <>
struct Logit<2> {  // fp32
    typedef uint32_t raw;
    static constexpr int KEY_SHIFT = 0;
    static constexpr uint32_t NOTHING = 0xff800000u;
    static __device__ __forceinline__ float value(uint32_t b) { return __uint_as_float(b); }
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }
    static __device__ __forceinline__ float larger(uint32_t a) { return __uint_as_float(a); }
    static constexpr uint32_t NOTHING2 = 0xff800000u;
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

// exp((x - top) / T) in fp32, 1 at the top; 0 or NaN where there is nothing to choose (-inf, NaN).
// The quotient is the IEEE one (ids must not depend on how it is computed): with y = 1 / T rounded once, two
// corrections q += (d - q T) y by fused multiply-adds round d / T correctly (P. Markstein, "Computation of
// elementary functions on the IBM RISC System/6000 processor", 1990), where nothing leaves the normal range.
struct Likelihood {
    float top, T, inv;
    bool plain;  // T far from 1 or an infinite top: the compiler's division, and the top's own case
    __device__ __forceinline__ void set(float top_, float T_) {
        top = top_;
        T = T_;
        inv = __frcp_rn(T_);
        plain = !(T_ > 1e-15f && T_ < 1e15f) || top_ == INFINITY;
    }
    // Loops over many values choose between the two outside: a branch a value keeps values from overlapping
    // (32 rows of 107,520 unfiltered: 14.3 us, so 12.6).
    __device__ __forceinline__ float operator()(float x) const { return plain ? slow(x) : quick(x); }
    __device__ __forceinline__ float slow(float x) const {
        return x == top && x > -INFINITY ? 1.f : expf(__fdiv_rn(x - top, T));
    }
    __device__ __forceinline__ float quick(float x) const {
        const float d = x - top;
        float q = d * inv;
        q = fmaf(fmaf(-q, T, d), inv, q);
        q = fmaf(fmaf(-q, T, d), inv, q);
        return expf(q);
    }
};
constexpr float LEAST = 9.094947017729282e-13f;  // 2^-40: anything less likely weighs nothing

// floor(2^40 e), 2^-40 <= e <= 1
__device__ __forceinline__ u64 fixed(float e) {
    const uint32_t b = __float_as_uint(e);
    return (u64((b & 0x7fffffu) | 0x800000u) << 17) >> (127u - (b >> 23));
}

// Sum of floor(2^40 e) over few thousand e <= 1 in two 32-bit words, without a 64-bit operation or a conversion an
// addend: adding 2^23 towards zero leaves the whole part of 2^20 e in the low mantissa bits, and what it cut off,
// times 2^20 the same way, the next 20 bits. The words add up the floats' bits; 2^23's own are taken out at the end.
struct WeightSum {
    uint32_t high = 0, low = 0, number = 0;
    static constexpr int MOST = 4095;  // addends: 4095 * 2^20 < 2^32
    __device__ __forceinline__ void add(float e) {
        const float x = e * 1048576.f, whole = __fadd_rz(x, 8388608.f);
        high += __float_as_uint(whole);
        low += __float_as_uint(__fmaf_rz(x - (whole - 8388608.f), 1048576.f, 8388608.f));
        number++;
    }
    __device__ __forceinline__ u64 total() const {
        const uint32_t ones = number * 0x4b000000u;
        return (u64(high - ones) << 20) + (low - ones);
    }
};

// fraction * total / 2^24 in whole numbers (fraction <= 2^24, total < 2^62), rounded down or up
__device__ __forceinline__ u64 share(u64 fraction, u64 total, bool up) {
    return fraction * (total >> 24) + ((fraction * (total & 0xffffffull) + (up ? 0xffffffull : 0ull)) >> 24);
}

// ln(w / total) from whole numbers: near 1 by what is missing, so that no digits cancel. Both sums, their quotient and the
// logarithm are rounded to fp32: below 2^-21 of the larger of the result and 1. In 64 bits, with one rounding, a
// call took 0.2 (one row: 7.9 us) to 0.5 us (32 rows of mixed controls: 15.6 us) more.
__device__ __forceinline__ float log_share(u64 w, u64 total) {
    if (2 * w > total) return log1pf(-__fdiv_rn(float(total - w), float(total)));
    return logf(__fdiv_rn(float(w), float(total)));
}

// In three parts whose sums over 32 lanes fit 32 bits (the upper one's wraps as the whole sum would): three
// independent reductions instead of five dependent exchanges of two words (0.3 to 0.5 us a call).
__device__ __forceinline__ u64 warp_add(u64 v) {
    const uint32_t low = __reduce_add_sync(FULL_MASK, uint32_t(v) & 0x7ffffffu);
    const uint32_t mid = __reduce_add_sync(FULL_MASK, uint32_t(v >> 27) & 0x7ffffffu);
    const uint32_t high = __reduce_add_sync(FULL_MASK, uint32_t(v >> 54));
    return (u64(high) << 54) + (u64(mid) << 27) + low;
}

// inclusive, in lane order
__device__ __forceinline__ u64 warp_scan(u64 v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 y = __shfl_up_sync(FULL_MASK, v, o);
        if ((threadIdx.x & 31) >= o) v += y;
    }
    return v;
}

struct Pair {
    u64 a, b;
};

struct Shared {
    u64 hist[2][BINS];  // two, used in turn: one may still be read by other blocks while the next fills
    Pair exchange[4][MAX_CLUSTER];  // likewise; [i][c] is written by block c
    static_assert(LIST == 2 * SAMPLE_THREADS && GROUPS * 4 == SAMPLE_THREADS, "two entries a thread, four threads a group");
    u64 list[LIST];     // ~key << 32 | id, so ascending order is what ties need; the first block's takes in all
    u64 inbox[LIST];    // of the first block: an equal share for every block of the cluster; later a shorter list
    uint32_t listed, counts[MAX_CLUSTER];
    uint32_t found;       // 16-byte packs of the slice that hold something for the list, and which
    uint16_t packs[LIST];
    static_assert(SLICE_BYTES / 16 <= 65536, "a pack's number fits 16 bits");
    u64 few[FEW], sorted[FEW];  // weights of listed ids, as listed and from the largest down
    static_assert(FEW == 4 * 32, "four a lane");
    float tops[GROUPS];  // the largest value of every group of threads
    float least_top;
    Pair warp_pairs[SAMPLE_WARPS];
    u64 scan[SAMPLE_WARPS];
    // a histogram's answer: the bin, the amount before it, the amount in it
    u64 bin, before, amount;
};

template <int TYPE>
struct Row {
    typedef typename Logit<TYPE>::raw raw;
    static constexpr int VEC = 16 / sizeof(raw), KS = Logit<TYPE>::KEY_SHIFT;
    cg::cluster_group cluster = cg::this_cluster();
    Shared& sh;
    raw* slice;           // the block's slice, `cached` values of it
    const raw* row;
    int vocab, rank, ranks;
    int lead;             // the row begins `lead` values after a 16-byte boundary: value j is id j - lead
    int begin, length, cached;  // the block's values [begin, begin + length)
    int mine0, mine1;     // this thread's values, from begin
    int turn = 0, hist_turn = 1;
    float top;
    Likelihood like;

    __device__ Row(Shared& s) : sh(s) {}

    __device__ __forceinline__ raw raw_at(int i) const {
        if (i < cached) return slice[i];
        const int id = begin + i - lead;
        return id >= 0 && id < vocab ? row[id] : Logit<TYPE>::NOTHING;
    }
    __device__ __forceinline__ float at(int i) const { return Logit<TYPE>::value(raw_at(i)); }
    // act(x, pure(x), i) for this thread's values in index order; four reads and four pure(x) are in flight
    // together, so that their latencies overlap.
    template <typename F, typename G>
    __device__ __forceinline__ void each(F pure, G act) const {
        constexpr int BATCH = 4;
        int i = mine0;
        for (const int end = min(mine1, cached); i + BATCH <= end; i += BATCH) {
            float x[BATCH];
            decltype(pure(0.f)) y[BATCH];
#pragma unroll
            for (int e = 0; e < BATCH; e++) x[e] = Logit<TYPE>::value(slice[i + e]);
#pragma unroll
            for (int e = 0; e < BATCH; e++) y[e] = pure(x[e]);
#pragma unroll
            for (int e = 0; e < BATCH; e++) act(x[e], y[e], i + e);
        }
        for (; i < mine1; i++) {
            const float x = at(i);
            act(x, pure(x), i);
        }
    }
    // act(pure(x)) for all of the block's values in no order, a pack of 16 bytes at a time (32 rows by top-p: 18.9 us,
    // value by value 0.5 more).
    template <typename F, typename G>
    __device__ __forceinline__ void each_pack(F pure, G act) const {
        const int packs = (cached + VEC - 1) / VEC;
        for (int p = threadIdx.x; p < packs; p += SAMPLE_THREADS) {
            __align__(16) raw x[VEC];
            *reinterpret_cast<uint4*>(x) = reinterpret_cast<const uint4*>(slice)[p];
            decltype(pure(0.f)) y[VEC];
#pragma unroll
            for (int e = 0; e < VEC; e++) y[e] = pure(Logit<TYPE>::value(x[e]));
#pragma unroll
            for (int e = 0; e < VEC; e++) act(y[e]);
        }
        for (int i = cached + threadIdx.x; i < length; i += SAMPLE_THREADS) act(pure(at(i)));
    }
    static __device__ __forceinline__ uint32_t key(float x) { return order_key(x) >> Logit<TYPE>::KEY_SHIFT; }

    __device__ __forceinline__ u64 weight(float x) const {
        const float e = like(x);
        return e >= LEAST ? fixed(e) : 0ull;
    }

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
        Pair* const places = sh.exchange[turn++ & 3];
        if (threadIdx.x < ranks) *cluster.map_shared_rank(places + rank, threadIdx.x) = block;
        cluster.sync();
        const int lane = threadIdx.x & 31;
        Pair p{0, 0};
        if (lane < ranks) p = places[lane];
        before.a = warp_add(lane < rank ? p.a : 0ull);
        before.b = warp_add(lane < rank ? p.b : 0ull);
        return Pair{warp_add(p.a), warp_add(p.b)};
    }
    // Exclusive running sum over the block in thread order.
    __device__ __forceinline__ u64 block_scan(u64 v) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        const u64 x = warp_scan(v);
        __syncthreads();
        if (lane == 31) sh.scan[warp] = x;
        __syncthreads();
        u64 before = 0;
#pragma unroll
        for (int w = 0; w < SAMPLE_WARPS; w++) before += w < warp ? sh.scan[w] : 0ull;
        return before + x - v;
    }

    // Histograms over the cluster, of numbers or of weights: cleared, filled by every block (larger values in
    // lower bins), and after a cluster barrier read by find().
    __device__ __forceinline__ void clear() {
        hist_turn++;
        if (threadIdx.x < BINS) sh.hist[hist_turn & 1][threadIdx.x] = 0;
        if (threadIdx.x == 0) sh.bin = BINS;
        __syncthreads();
    }
    template <bool WEIGHTS>
    __device__ __forceinline__ void put(int bin, u64 w) {
        u64* const at = sh.hist[hist_turn & 1] + bin;
        if (WEIGHTS) atomicAdd(at, w);
        else atomicAdd(reinterpret_cast<uint32_t*>(at), 1u);  // below 2^32: the lower half is enough
    }
    // The first bin at which `base` and the amounts up to it reach `need` (left in sh.bin / before / amount); false
    // when they do not.
    __device__ __forceinline__ bool find(u64 base, u64 need) {
        u64 sum = 0;
        if (threadIdx.x < BINS) {
#pragma unroll
            for (int c = 0; c < MAX_CLUSTER; c++)  // all reads in flight together
                if (c < ranks) sum += cluster.map_shared_rank(sh.hist[hist_turn & 1], c)[threadIdx.x];
        }
        const u64 before = base + block_scan(sum);
        if (before < need && need <= before + sum) {
            sh.bin = threadIdx.x;
            sh.before = before;
            sh.amount = sum;
        }
        __syncthreads();
        return sh.bin < BINS;
    }
    // All three; classify(x) gives a value's bin or -1.
    template <bool WEIGHTS, typename F>
    __device__ __forceinline__ bool histogram(F classify, u64 base, u64 need) {
        clear();
        each(classify, [&](float x, int bin, int) {
            const u64 w = WEIGHTS && bin >= 0 ? weight(x) : 1ull;
            if (bin >= 0 && w) put<WEIGHTS>(bin, w);
        });
        cluster.sync();
        return find(base, need);
    }

    // Steps of (max - x) up to `limit` below the largest; -1 beyond it.
    struct Steps {
        float top, limit, step;
        __device__ __forceinline__ int operator()(float x) const {
            const float d = top - x;
            if (!(x > -INFINITY) || d > limit) return -1;
            return min(int(d * step), BINS - 1);
        }
        // bounds of the values in a bin, wider than the two roundings above
        __device__ __forceinline__ float largest(int bin) const {
            return __double2float_ru(double(top) - (bin ? bin / double(step) : 0.0) * (1.0 - 1e-6));
        }
        __device__ __forceinline__ float least(int bin) const {
            if (top == INFINITY) return top;
            return __double2float_rd(double(top) - (bin == BINS - 1 ? double(limit) : (bin + 1) / double(step)) * (1.0 + 1e-6));
        }
    };

    // Lists this block's values x >= from, down to `far` below the top. Few are: packs of 16 bytes are looked through
    // by their largest value first, and the found packs then value by value (32 rows of 107,520 by top-k 11.0 us, by top-p
    // 18.9; value by value from the start 1.8 more).
    __device__ __forceinline__ void list_from(float from, float far) {
        if (threadIdx.x == 0) sh.listed = sh.found = 0;
        __syncthreads();
        auto wanted = [&](float x) { return x >= from && x > -INFINITY && !(top - x > far); };
        auto put_in = [&](float x, int i) {
            const uint32_t n = atomicAdd(&sh.listed, 1u);
            if (n < LIST) sh.list[n] = u64(~key(x)) << 32 | uint32_t(begin + i - lead);
        };
        const int packs = (cached + VEC - 1) / VEC;  // the last one is filled up with NOTHING
        for (int p = threadIdx.x; p < packs; p += SAMPLE_THREADS) {
            const uint4 v = reinterpret_cast<const uint4*>(slice)[p];
            if (!wanted(Logit<TYPE>::larger(Logit<TYPE>::max2(Logit<TYPE>::max2(v.x, v.y), Logit<TYPE>::max2(v.z, v.w))))) continue;
            const uint32_t n = atomicAdd(&sh.found, 1u);
            if (n < LIST) sh.packs[n] = uint16_t(p);
            else atomicMax(&sh.listed, LIST + 1u);  // each holds one for the list at least: too many
        }
        for (int i = cached + threadIdx.x; i < length; i += SAMPLE_THREADS)
            if (const float x = at(i); wanted(x)) put_in(x, i);
        __syncthreads();
        const int values = int(min(sh.found, uint32_t(LIST))) * VEC;
        for (int j = threadIdx.x; j < values; j += SAMPLE_THREADS) {
            const int i = sh.packs[j / VEC] * VEC + j % VEC;
            if (const float x = Logit<TYPE>::value(slice[i]); wanted(x)) put_in(x, i);
        }
    }
    // Brings the blocks' lists together in the first block; the number of ids, or -1 when they do not fit. Each block
    // leaves up to its share in the first block's inbox before the barrier that makes the numbers known; only when
    // some block has more does it take a second barrier. Two sums over the cluster travel along.
    __device__ __forceinline__ int deliver(Pair& sums) {
        __syncthreads();
        const uint32_t mine = sh.listed, share = LIST / ranks;
        if (rank) {
            u64* const to = cluster.map_shared_rank(sh.inbox, 0) + rank * share;
            for (uint32_t i = threadIdx.x; i < min(mine, share); i += SAMPLE_THREADS) to[i] = sh.list[i];
        }
        if (threadIdx.x < ranks) *cluster.map_shared_rank(sh.counts + rank, threadIdx.x) = mine;
        Pair unused;
        sums = exchange(sums, unused);
        // thread t takes what block t / TEAM has brought, all blocks' together
        constexpr int TEAM = SAMPLE_THREADS / MAX_CLUSTER;
        const int giver = threadIdx.x / TEAM;
        uint32_t total = 0, before = 0, at = 0;
        bool over = false;
#pragma unroll
        for (int c = 0; c < MAX_CLUSTER; c++) {
            const uint32_t n = c < ranks ? sh.counts[c] : 0u;
            over |= n > share;
            before += c < rank ? n : 0u;
            at += c < giver ? n : 0u;
            total += n;
        }
        if (total > LIST) return -1;
        if (over) {
            if (rank) {
                u64* const to = cluster.map_shared_rank(sh.list, 0) + before;
                for (uint32_t i = threadIdx.x; i < mine; i += SAMPLE_THREADS) to[i] = sh.list[i];
            }
            cluster.sync();
        } else if (rank == 0) {
            if (giver > 0 && giver < ranks)
                for (uint32_t i = threadIdx.x % TEAM; i < sh.counts[giver]; i += TEAM) sh.list[at + i] = sh.inbox[giver * share + i];
            __syncthreads();
        }
        return int(total);
    }
    // Both.
    __device__ __forceinline__ int gather(float from, float far) {
        list_from(from, far);
        Pair none{0, 0};
        return deliver(none);
    }

    // Sorts the list's first n entries ascending (n a power of two): bitonic, in shared memory.
    __device__ __forceinline__ void sort_list(u64* list, int n) {
        for (int size = 2; size <= n; size *= 2)
            for (int gap = size / 2; gap > 0; gap /= 2) {
                __syncthreads();
                if (threadIdx.x < n / 2) {
                    const int i = threadIdx.x, lo = 2 * i - (i & (gap - 1)), hi = lo + gap;
                    const u64 a = list[lo], b = list[hi];
                    if ((a > b) == ((lo & size) == 0)) {
                        list[lo] = b;
                        list[hi] = a;
                    }
                }
            }
        __syncthreads();
    }

    // The row's last steps, by the first block alone: n ids on the list hold everything that can be kept. run_known: the
    // weight that top-p is a share of (0: that of the first k listed ones).
    __device__ __forceinline__ void finish_list(const SampleArgs& a, int r, int n, int k, u64 p24, u64 least, u64 m, u64 run_known) {
        if (rank != 0) return;
        u64* list = sh.list;
        const bool nucleus = p24 < (1ull << 24);
        if (n > FEW && (k < n || (nucleus && run_known))) {
            // a shorter list: the values up to the step where k, or p, is reached
            const Steps steps{top, like.T * SPAN, float(BINS) / (like.T * SPAN)};
            clear();
            if (threadIdx.x == 0) sh.listed = 0;
            for (int i = threadIdx.x; i < n; i += SAMPLE_THREADS) {
                const float x = key_value<KS>(uint32_t(~list[i] >> 32));
                const u64 w = k < n ? 1ull : weight(x);
                if (!w) continue;
                // 20 bits each: at most 1024 ids, so neither sum leaves 32 bits
                uint32_t* const bin = reinterpret_cast<uint32_t*>(sh.hist[hist_turn & 1] + steps(x));
                atomicAdd(bin, uint32_t(w) & 0xfffffu);
                if (w >> 20) atomicAdd(bin + 1, uint32_t(w >> 20));
            }
            __syncthreads();
            const u64 need = k < n ? u64(k) : max(share(p24, run_known, true), 1ull);
            const uint32_t* const bin = reinterpret_cast<const uint32_t*>(sh.hist[hist_turn & 1] + threadIdx.x % BINS);
            const u64 sum = threadIdx.x < BINS ? (u64(bin[1]) << 20) + bin[0] : 0ull, before = block_scan(sum);
            if (before < need && need <= before + sum) sh.bin = threadIdx.x;
            __syncthreads();
            for (int i = threadIdx.x; i < n; i += SAMPLE_THREADS) {
                const u64 entry = list[i];
                if (u64(steps(key_value<KS>(uint32_t(~entry >> 32)))) <= sh.bin) sh.inbox[atomicAdd(&sh.listed, 1u)] = entry;
            }
            __syncthreads();
            list = sh.inbox;
            n = int(sh.listed);
        }
        if (n <= FEW) finish_few(list, a, r, n, k, p24, least, m, run_known);
        else finish_many(list, a, r, n, k, p24, least, m, run_known);
    }
    // By sorting, two neighbouring entries a thread.
    __device__ __forceinline__ void finish_many(u64* list, const SampleArgs& a, int r, int n, int k, u64 p24, u64 least, u64 m,
                                                u64 run_known) {
        const int t = threadIdx.x;
        int size = 2;
        while (size < n) size *= 2;
        for (int i = n + t; i < size; i += SAMPLE_THREADS) list[i] = ~0ull;
        sort_list(list, size);
        u64 w[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int i = 2 * t + e;
            w[e] = i < n && i < k ? weight(key_value<KS>(uint32_t(~list[i] >> 32))) : 0ull;
        }
        const u64 before = block_scan(w[0] + w[1]);
        if (p24 < (1ull << 24)) {
            const u64 run = run_known ? run_known : block_add({w[0] + w[1], 0}).a, need = max(share(p24, run, true), 1ull);
            if (before + w[0] >= need) w[1] = 0;
            if (before >= need) w[0] = 0;
        }
        if (w[0] < least) w[0] = 0;
        if (w[1] < least) w[1] = 0;
        const Pair total = block_add({w[0] + w[1], u64((w[0] != 0) + (w[1] != 0))});
        // the kept ones are the first total.b; now in index order, each with its key
        const int kept = int(total.b);
        size = 2;
        while (size < kept) size *= 2;
        u64 entry[2];
#pragma unroll
        for (int e = 0; e < 2; e++) entry[e] = 2 * t + e < kept ? list[2 * t + e] : 0ull;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 2; e++)
            if (2 * t + e < size) list[2 * t + e] = 2 * t + e < kept ? entry[e] << 32 | uint32_t(~entry[e] >> 32) : ~0ull;
        sort_list(list, size);
#pragma unroll
        for (int e = 0; e < 2; e++) w[e] = 2 * t + e < kept ? weight(key_value<KS>(uint32_t(list[2 * t + e]))) : 0ull;
        const u64 target = share(m, total.a, false);
        u64 upto = block_scan(w[0] + w[1]);
#pragma unroll
        for (int e = 0; e < 2; e++) {
            if (upto <= target && target < upto + w[e]) {
                a.ids[r] = int(list[2 * t + e] >> 32);
                if (a.logprobs) a.logprobs[r] = log_share(w[e], total.a);
            }
            upto += w[e];
        }
        if (t == 0 && a.kept) a.kept[r] = kept;
    }
    // Places and running weights of at most FEW ids by comparing each with each, four threads (or eight) an id: fewer
    // dependent steps than a sort. What top-p leaves is found by each warp for itself, from all weights in order (with
    // sums over the block instead, 1 to 2 us more).
    __device__ __forceinline__ void finish_few(const u64* list, const SampleArgs& a, int r, int n, int k, u64 p24, u64 least, u64 m,
                                               u64 run_known) {
        const int team = n <= FEW / 2 ? 8 : 4, i = threadIdx.x / team, part = threadIdx.x % team;
        const u64 mine = i < n ? list[i] : ~0ull;
        auto team_add = [&](auto v) {
            for (int o = 1; o < team; o *= 2) v += __shfl_xor_sync(FULL_MASK, v, o);
            return v;
        };
        uint32_t place = 0;
#pragma unroll 8
        for (int j = part; j < n; j += team) place += list[j] < mine;
        place = team_add(place);
        u64 w = i < n && place < uint32_t(k) ? weight(key_value<KS>(uint32_t(~mine >> 32))) : 0ull;
        if (part == 0 && i < n) sh.sorted[place] = w;
        __syncthreads();
        // every warp by itself: the weights in order, four a lane, and what top-p and min-p leave of them
        const int lane = threadIdx.x & 31;
        u64 x[4], sum = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) sum += x[e] = 4 * lane + e < n ? sh.sorted[4 * lane + e] : 0ull;
        if (p24 < (1ull << 24)) {
            const u64 upto = warp_scan(sum), run = run_known ? run_known : __shfl_sync(FULL_MASK, upto, 31);
            const u64 need = max(share(p24, run, true), 1ull);
            u64 before = upto - sum;
            uint32_t within = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const u64 y = x[e];
                if (before < need) within++;
                else x[e] = 0;
                before += y;
            }
            if (place >= __reduce_add_sync(FULL_MASK, within)) w = 0;
        }
        if (w < least) w = 0;
        if (part == 0 && i < FEW) sh.few[i] = w;
        sum = 0;
        uint32_t some = 0;
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (x[e] >= least) {
                sum += x[e];
                some++;
            }
        const Pair total{warp_add(sum), __reduce_add_sync(FULL_MASK, some)};
        __syncthreads();
        const u64 target = share(m, total.a, false);
        u64 upto = 0;  // kept weight of the lower ids
#pragma unroll 8
        for (int j = part; j < n; j += team) upto += uint32_t(list[j]) < uint32_t(mine) ? sh.few[j] : 0ull;
        upto = team_add(upto);
        if (part == 0 && upto <= target && target < upto + w) {
            a.ids[r] = int(uint32_t(mine));
            if (a.logprobs) a.logprobs[r] = log_share(w, total.a);
        }
        if (threadIdx.x == 0 && a.kept) a.kept[r] = int(total.b);
    }

    // After histogram() over `steps`: the key at which the amounts of the values, from the largest down, reach
    // `need`; before and amount: the amounts above it and at it.
    template <bool WEIGHTS>
    __device__ __forceinline__ void narrow(const Steps& steps, u64 need, uint32_t least_key, uint32_t& edge, u64& before,
                                           u64& amount) {
        const int bin = int(sh.bin);
        u64 base = sh.before;
        uint32_t khi = key(steps.largest(bin)), klo = key(steps.least(bin));
        while (true) {
            const int bits = 32 - __clz(khi - klo), shift = max(bits - 8, 0);
            __syncthreads();  // the answer before has been read
            auto fine = [&](float x) -> int {
                const uint32_t k = key(x);
                return k < least_key || k > khi || k < klo || steps(x) != bin ? -1 : int((khi - k) >> shift);
            };
            histogram<WEIGHTS>(fine, base, need);
            base = sh.before;
            khi -= uint32_t(sh.bin) << shift;
            if (!shift) break;
            klo = max(klo, khi - ((1u << shift) - 1u));
        }
        edge = khi;
        before = base;
        amount = sh.amount;
        __syncthreads();
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
    row.cluster.barrier_arrive();  // waited for before the first access to another block's shared memory
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
    static_assert(SAMPLE_MAX_VOCAB / MAX_CLUSTER / SAMPLE_THREADS + 1 <= WeightSum::MOST, "a thread's weights fit their sums");
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

    // read the slice once; the largest logit
    uint32_t top2 = Logit<TYPE>::NOTHING2;
    constexpr int BATCH = 4;  // reads in flight together
    for (int v0 = t; v0 * VEC < row.length; v0 += BATCH * SAMPLE_THREADS) {
        uint4 x4[BATCH];
#pragma unroll
        for (int b = 0; b < BATCH; b++) {
            const int j = (v0 + b * SAMPLE_THREADS) * VEC, id = row.begin + j - row.lead;
            if (j < row.length && id >= 0 && id + VEC <= V) {
                x4[b] = __ldg(reinterpret_cast<const uint4*>(row.row + id));
            } else {  // the row's ends
                raw x[VEC];
#pragma unroll
                for (int e = 0; e < VEC; e++)
                    x[e] = j < row.length && id + e >= 0 && id + e < V ? row.row[id + e] : Logit<TYPE>::NOTHING;
                x4[b] = *reinterpret_cast<const uint4*>(x);
            }
        }
#pragma unroll
        for (int b = 0; b < BATCH; b++) {
            const int j = (v0 + b * SAMPLE_THREADS) * VEC;
            if (j < row.cached) *reinterpret_cast<uint4*>(row.slice + j) = x4[b];
            const uint32_t pairs[4] = {x4[b].x, x4[b].y, x4[b].z, x4[b].w};
#pragma unroll
            for (int e = 0; e < 4; e++) top2 = Logit<TYPE>::max2(top2, pairs[e]);
        }
    }
    const int lanes = 4 * row.ranks;  // of a group
    float top = Logit<TYPE>::larger(top2);
    for (int o = 1; o < lanes; o *= 2) top = fmaxf(top, __shfl_xor_sync(FULL_MASK, top, o));
    row.cluster.barrier_wait();
    // every group's largest value to every block: lane c of a group (it has at least as many) writes to block c
    if (t % lanes < row.ranks)
        row.cluster.map_shared_rank(shared.tops, t % lanes)[(row.rank * SAMPLE_THREADS + t) / lanes] = top;
    row.cluster.sync();
    for (int i = t & 31; i < GROUPS; i += 32) top = fmaxf(top, shared.tops[i]);
    top = warp_max(top);
    row.top = top;
    row.like.set(top, T);

    const float far = SPAN * T;
    const u64 m = u > 0.f ? min(u64(fminf(u, 1.f) * 16777216.0f), (1ull << 24) - 1) : 0ull;
    const bool nucleus = p24 < (1ull << 24);
    typedef typename Row<TYPE>::Steps Steps;
    constexpr int KS = Logit<TYPE>::KEY_SHIFT;

    if (k < V && V <= LIST) {  // all of them
        const int n = row.gather(-INFINITY, far);
        if (n > 0) {
            row.finish_list(a, r, n, k, p24, least, m, 0);
            return;
        }
    }
    // kept: keys above `edge`, and the first `ties` (in index order) of the `at_edge` values at it
    uint32_t edge = 0;
    u64 ties = 0, at_edge = 0, before, amount;
    if (k <= 2 * GROUPS) {
        const int some = __syncthreads_count(t < GROUPS && shared.tops[t % GROUPS] > -INFINITY);  // groups that have a value
        const int wanted = k <= GROUPS / 2 ? k : int(ceilf(GROUPS * (1.f - __expf(-(1.25f * k + 24.f) / GROUPS))));
        const int j = max(min(wanted, some), 1);
        // the j-th largest of the groups' maxima: a quarter of them for each of four threads to compare with
        const float own = shared.tops[t / 4];
        int above = 0, no_less = 0;
#pragma unroll 8
        for (int o = t & 3; o < GROUPS; o += 4) {
            above += shared.tops[o] > own;
            no_less += shared.tops[o] >= own;
        }
        above += __shfl_xor_sync(FULL_MASK, above, 1);
        no_less += __shfl_xor_sync(FULL_MASK, no_less, 1);
        above += __shfl_xor_sync(FULL_MASK, above, 2);
        no_less += __shfl_xor_sync(FULL_MASK, no_less, 2);
        if (above < j && j <= no_less) shared.least_top = own;  // equal maxima write the same
        __syncthreads();
        const float from = shared.least_top;
        const int n = row.gather(from, far);
        // fewer than k are enough where none of the others weighs anything: nothing further down was left out
        if (n >= k || (n > 0 && (from == -INFINITY || top - from > far))) {
            row.finish_list(a, r, n, k, p24, least, m, 0);
            return;
        }
    }
    if (k < V) {
        const Steps steps{top, far, float(BINS) / far};
        if (row.template histogram<false>(steps, 0, k)) {
            const int n = shared.before + shared.amount <= LIST ? row.gather(steps.least(int(shared.bin)), far) : -1;
            if (n >= 0) {
                row.finish_list(a, r, n, k, p24, least, m, 0);
                return;
            }
            row.template narrow<false>(steps, k, 0u, edge, before, amount);
            at_edge = amount;
            ties = k - before;
        }
    }
    if (nucleus) {
        // all weights; then a list of the values near the top, and what those weigh (a pass of its own: filling the
        // list inside the first one made its loop so long that it took twice the time)
        WeightSum all_weight;
        auto add = [&](float e) { all_weight.add(e >= LEAST ? e : 0.f); };
        if (edge) row.each_pack([&](float x) { return x > -INFINITY && row.key(x) >= edge ? row.like(x) : 0.f; }, add);
        else if (row.like.plain) row.each_pack([&](float x) { return row.like.slow(x); }, add);
        else row.each_pack([&](float x) { return row.like.quick(x); }, add);
        const float near = far * 0.3f;
        row.list_from(edge ? key_value<KS>(edge) : -INFINITY, near);
        __syncthreads();
        u64 near_weight = 0;
        for (int i = t; i < min(int(shared.listed), LIST); i += SAMPLE_THREADS)
            near_weight += row.weight(key_value<KS>(uint32_t(~shared.list[i] >> 32)));
        Pair sums = row.block_add({all_weight.total(), near_weight});
        const int n = row.deliver(sums);
        const u64 cut_off = ties < at_edge ? (at_edge - ties) * row.weight(key_value<KS>(edge)) : 0ull;
        const u64 run = sums.a - cut_off, need = max(share(p24, run, true), 1ull);
        if (n >= 0 && run && sums.b >= need && !cut_off) {
            row.finish_list(a, r, n, k, p24, least, m, run);
            return;
        }
        // an id whose weight V times over fits into what may be left out is left out itself
        const u64 small = (run - min(need, run)) / u64(V);
        const float limit = small > 1 ? fminf(far, T * (log2f(1099511627776.0f / float(small)) * 0.6931472f) * 1.0001f + 1e-6f * T) : far;
        const Steps steps{top, limit, float(BINS) / limit};
        auto within = [&](float x) -> int { return row.key(x) < edge ? -1 : steps(x); };
        const bool found = run && row.template histogram<true>(within, 0, need);
        if (found) {
            if (ties == at_edge) {  // top-k has not cut through equal values
                const float from = steps.least(int(shared.bin));
                const int n = row.gather(edge ? fmaxf(from, key_value<KS>(edge)) : from, far);
                if (n >= 0) {
                    row.finish_list(a, r, n, k, p24, least, m, run);
                    return;
                }
            }
            uint32_t cut = edge;
            row.template narrow<true>(steps, need, edge, cut, before, amount);
            const u64 each = row.weight(key_value<KS>(cut));
            ties = (need - before + each - 1) / each;
            at_edge = amount / each;
            edge = cut;
        }
    }
    // ranks of the values at the edge, where only some of them are kept
    u64 first_tie = 0;
    if (ties < at_edge) {
        u64 n = 0;
        row.each([&](float x) { return x > -INFINITY && row.key(x) == edge; }, [&](float, bool at, int) { n += at; });
        Pair ahead;
        row.exchange(row.block_add({n, 0}), ahead);
        first_tie = ahead.a + row.block_scan(n);
    }
    // w >= least, both whole, is e >= least / 2^40: exact in fp32, min_p having 24 bits
    const float least_e = float(least) * LEAST;
    const uint32_t tie_end = ties < at_edge ? uint32_t(ties) : 0xffffffffu;
    WeightSum sum;
    uint32_t my_count = 0, tie = uint32_t(first_tie);
    auto add = [&](float e) {
        const bool kept = e >= least_e;
        sum.add(kept ? e : 0.f);
        my_count += kept;
    };
    if (edge) {
        row.each([&](float x) { return x > -INFINITY ? row.key(x) : 0u; },
                 [&](float x, uint32_t key, int) {
                     if (key > edge || (key == edge && tie++ < tie_end)) add(row.like(x));
                 });
    } else {
        auto put = [&](float, float e, int) { add(e); };
        if (row.like.plain) row.each([&](float x) { return row.like.slow(x); }, put);
        else row.each([&](float x) { return row.like.quick(x); }, put);
    }
    const u64 my_weight = sum.total();
    Pair ahead;
    const Pair total = row.exchange(row.block_add({my_weight, my_count}), ahead);
    const u64 target = share(m, total.a, false);
    const u64 upto = ahead.a + row.block_scan(my_weight);
    // the thread whose values hold the target: its warp looks through them, a value a lane
    const unsigned holds = __ballot_sync(FULL_MASK, upto <= target && target < upto + my_weight);
    if (holds) {
        const int owner = __ffs(holds) - 1, lane = t & 31;
        const int i1 = __shfl_sync(FULL_MASK, row.mine1, owner);
        u64 run = __shfl_sync(FULL_MASK, upto, owner);
        uint32_t seen = __shfl_sync(FULL_MASK, uint32_t(first_tie), owner);
        for (int i0 = __shfl_sync(FULL_MASK, row.mine0, owner); i0 < i1; i0 += 32) {
            const int i = i0 + lane;
            const float x = i < i1 ? row.at(i) : -INFINITY;
            const uint32_t key = row.key(x);
            const unsigned equal = __ballot_sync(FULL_MASK, x > -INFINITY && edge && key == edge);
            const bool in = x > -INFINITY && (key > edge || !edge || (key == edge && seen + __popc(equal & ((1u << lane) - 1u)) < tie_end));
            seen += __popc(equal);
            const float e = row.like(x);
            const u64 w = in && e >= least_e ? fixed(e) : 0ull;
            const u64 incl = warp_scan(w);
            const unsigned past = __ballot_sync(FULL_MASK, target < run + incl);
            if (past) {
                if (lane == __ffs(past) - 1) {
                    a.ids[r] = row.begin + i - row.lead;
                    if (a.logprobs) a.logprobs[r] = log_share(w, total.a);
                }
                break;
            }
            run += __shfl_sync(FULL_MASK, incl, 31);
        }
    }
    if (row.rank == 0 && t == 0) {
        if (a.kept) a.kept[r] = int(total.b);
        if (!total.a) {
            a.ids[r] = 0;
            if (a.logprobs) a.logprobs[r] = -INFINITY;
        }
    }
    // no block reads another's shared memory after the last exchange, so each may leave by itself
}

template <int TYPE>
cudaError_t launch(const SampleArgs& a, cudaStream_t s) {
    constexpr int SIZE = TYPE == 2 ? 4 : 2, VEC = 16 / SIZE;
    // blocks a row: enough that two blocks' slices fit an SM, and more while every block still has an SM of its own (32
    // rows of 107,520 by top-k: 11.0 us on 4 blocks a row, 5 more on 8, which share SMs)
    int ranks = 1;
    while (ranks < MAX_CLUSTER && a.vocab / ranks > 2048 &&
           ((long long)a.vocab * SIZE > (long long)ranks * (SLICE_BYTES / 4 * 3) || a.rows * ranks <= 74))
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
