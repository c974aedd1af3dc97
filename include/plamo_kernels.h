/* libplamo_cuda kernel-level entry points: the hot-path kernels on caller-provided DEVICE
 * buffers, enqueued on `stream` (a cudaStream_t, NULL = default stream). They return 0 on a
 * successful launch, non-zero with plamo_last_error() set otherwise; completion is the caller's
 * stream synchronisation. bf16 values are passed as uint16_t bit patterns. Each entry point names
 * the reference Metal kernel it replaces (Sources/Plamo/Kernels.metal, Batch.metal).
 */
#ifndef PLAMO_KERNELS_H
#define PLAMO_KERNELS_H

#include <stddef.h>
#include <stdint.h>

#ifndef PLAMO_API
#define PLAMO_API __attribute__((visibility("default")))
#endif

#ifdef __cplusplus
extern "C" {
#endif

/* linear (Kernels.metal:92-114), matrix (:149-200), project3/4 (Batch.metal:171-221).
 * y[r][m] = bf16(sum_k W[m][k] * x[r][k]) for r < rows, fp32 accumulation.
 * W: raw bf16 [M][K] (offsets == NULL), or a .p12 tensor: `w` = data region, `offsets` = tagged
 * block table (packed_four, Kernels.metal:33-44). K % 128 == 0.
 * mode 0: plain, y is [rows][M]. mode 1: SwiGLU epilogue (Kernels.metal:202-210): W has 2F rows,
 * y is [rows][F] = bf16(bf16(silu(g)) * u). mode 2: logits + first-index argmax
 * (Kernels.metal:704-729): y is [rows][M] bf16 logits and argmax_keys[r] (zeroed by the caller)
 * receives a 64-bit key, decoded by plamo_k_argmax_keys. */
PLAMO_API int plamo_k_linear(const void* w, const uint32_t* offsets, const uint16_t* x, int rows, int K, int M, int mode,
                   uint16_t* y, uint64_t* argmax_keys, void* stream);

/* The same projection on the tensor cores (tcgen05 GEMM, fp32 accumulation in tensor memory):
 * raw bf16 weights only (offsets are not taken), K a multiple of 64, any rows >= 1. The outputs
 * match plamo_k_linear within the rounding of the accumulation order. splits > 0 forces a K split
 * over that many CTAs per tile (<= 16 and <= K / 64), whose fp32 partials need
 * splits * rows * M floats of `workspace`; splits == 0 lets the launcher choose, splitting only
 * into the workspace given (workspace may then be NULL). */
PLAMO_API int plamo_k_linear_tc(const void* w, const uint16_t* x, int rows, int K, int M, int mode, uint16_t* y,
                                uint64_t* argmax_keys, int splits, float* workspace, size_t workspace_floats,
                                void* stream);

/* Sampler.select on caller-owned device buffers: logits [V] bf16, history [n] ids, scratch counts
 * [V] int32 and flags [V] bytes (cleared by the call); key_out receives the winning argmax key
 * (0 when no value is above -inf: the selected id is then 0, else 0xFFFFFFFF - low 32 bits).
 * Same semantics as plamo_select. */
PLAMO_API int plamo_k_select(const uint16_t* logits, int V, const int32_t* history, int n, float penalty,
                             int no_repeat_ngram, float frequency, float presence, int32_t* counts, uint8_t* flags,
                             uint64_t* key_out, void* stream);

/* Converts argmax keys to indices (0xFFFFFFFF when a row had only NaN). */
PLAMO_API int plamo_k_argmax_keys(const uint64_t* keys, int rows, uint32_t* out, void* stream);

/* norm (Kernels.metal:46-90): z = bf(bf(src*rsqrt(mean(src^2)+1e-6)) * bf(w+offset)).
 * residual == 0: x := z. residual != 0: x := bf(x + z) and, when next_w != NULL,
 * next := norm(x, next_w, offset 1). Rows of n <= 4096 values. */
PLAMO_API int plamo_k_norm(const uint16_t* w, const uint16_t* src, uint16_t* x, int rows, int n, float offset, int residual,
                 const uint16_t* next_w, uint16_t* next, void* stream);

/* argmax (Kernels.metal:704-729) over `rows` rows of n bf16 logits: first index of the maximum,
 * NaN never wins, all-NaN rows give 0xFFFFFFFF. `scratch` holds rows 64-bit keys. */
PLAMO_API int plamo_k_argmax(const uint16_t* logits, int rows, int n, uint64_t* scratch, uint32_t* out, void* stream);

/* packed_bits / packed_four (Kernels.metal:23-44): reconstructs `count` bf16 weights (count %
 * 16 == 0) from a .p12 data region and its tagged block table. */
PLAMO_API int plamo_k_packed_decode(const uint8_t* data, const uint32_t* entries, long long count, uint16_t* out, void* stream);

/* Split-K decode attention for one query row (attention + attention_merge, Kernels.metal:440-562;
 * matrix_rotary / softmax / attend, :301-437): q is heads*128 bf16 (already rotated);
 * keys/values are [cap][kv_heads][128] bf16. Keys r in [0,count) sit at slot (first + r) % cap;
 * the row sees r in [begin, end). Local layers (full == 0) re-rotate raw keys with coordinate r
 * using rope_local ([rows][64] u32 = cos bits | sin bits << 16). out: heads*128 bf16.
 * `splits` key partitions; the partial results live in library-owned device scratch that is
 * allocated on the first call and grown as needed (cudaMalloc). */
PLAMO_API int plamo_k_attention(const uint16_t* q, const uint16_t* keys, const uint16_t* values, int heads, int kv_heads,
                      int cap, int first, int count, int begin, int end, int full, const uint32_t* rope_local,
                      int splits, uint16_t* out, void* stream);

/* Attention of `rows` query rows over one cache (the prefill form of the split-K attention above,
 * Kernels.metal:301-562): q is [rows][heads*128] bf16 (already rotated); geo is a DEVICE array of
 * [rows][4] int32 {first, count, begin, end} per row as in plamo_k_attention (keys r in [0,count)
 * at slot (first + r) % cap, the row sees r in [begin, end)). tensor == 0: the CUDA-core kernels
 * with `splits` key partitions (bit-identical to the runtime's default path); tensor == 1: the
 * tcgen05 kernel of tensor mode's prefill (16 query heads over one KV head, splits chosen by the
 * library); tensor == 2: tensor mode's decode-row kernel (16 query heads over one KV head, warp-level
 * MMAs, the same `splits` as tensor == 0). 1 and 2 are within rounding of 0. Rows of one 16-token
 * chunk should be consecutive for tensor == 1; rows with
 * different windows are handled, at a lower rate. `workspace` (device, 256-byte aligned) holds the
 * row descriptors and split partials; a call that finds it too small fails with the bytes needed. */
PLAMO_API int plamo_k_attention_rows(const uint16_t* q, const uint16_t* keys, const uint16_t* values, int heads,
                                     int kv_heads, int cap, const int32_t* geo, int rows, int full,
                                     const uint32_t* rope_local, int splits, int tensor, uint16_t* out, void* workspace,
                                     size_t workspace_bytes, void* stream);

/* plamo_k_attention without any device allocation. No counterpart in the reference (whose Metal
 * encoder owns its buffers); for callers that must not allocate device memory during a call, such
 * as a serving loop that reserved its memory up front and can afford neither an out-of-memory
 * failure mid-stream nor the device-wide wait of the cudaFree with which plamo_k_attention grows
 * its scratch. Same arguments and results as plamo_k_attention. The partial results live in one
 * fixed 2 MiB device array per device (splits x heads at most 4032; larger requests fail with an
 * error and launch nothing). The first call on a device looks the array up (cudaGetSymbolAddress,
 * with that device current): make it before any stream capture. The address is kept for the life
 * of the process, so a device reset (cudaDeviceReset) in between invalidates it: do not call this
 * entry point on a device after resetting that device. Calls are asynchronous on
 * `stream` (they return once enqueued) and all calls on a device share the array, which keeps the
 * last call's contents: calls whose execution may overlap (other streams, other threads) race. */
PLAMO_API int plamo_k_attention_static(const uint16_t* q, const uint16_t* keys, const uint16_t* values, int heads,
                                       int kv_heads, int cap, int first, int count, int begin, int end, int full,
                                       const uint32_t* rope_local, int splits, uint16_t* out, void* stream);

/* The fp32 exponential used by the softmax and SwiGLU kernels (Kernels.metal:209, :386 use exp):
 * y[i] = e^x[i] from IEEE operations only (Cody-Waite reduction, degree-7 Taylor polynomial), so a
 * CPU restatement reproduces it exactly. n floats, device pointers. */
PLAMO_API int plamo_k_exp(const float* x, float* y, long long n, void* stream);

/* ---- A serving step over a paged key-value cache -------------------------------------------------
 * No counterpart in the reference, whose caches are one contiguous slab per lane (Batch.swift:33-78).
 * One step of a changing set of requests is
 *     plamo_k_paged_plan -> per layer: plamo_k_paged_qkv, plamo_k_paged_attention -> plamo_k_sample
 * All four enqueue on `stream`, allocate nothing, keep nothing between calls and can be captured in a
 * CUDA graph. Values are bf16 (dtype 0) or fp16 (dtype 1) bit patterns. Arrays of 32-bit values are 4-byte aligned. */

/* One layer's paged cache. The value of token slot t = page * page_size + offset, KV head h, element d
 * is at keys[page * page_stride + offset * token_stride + h * head_stride + d] (values alike); strides in
 * elements, multiples of 8, keys and values 16-byte aligned. head_dim 64 or 128; page_size >= 1. */
typedef struct plamo_paged_cache {
    void* keys;
    void* values;
    int32_t dtype;
    int32_t pages;
    int32_t page_size;
    int32_t kv_heads;
    int32_t head_dim;
    int64_t page_stride;
    int64_t token_stride;
    int64_t head_stride;
} plamo_paged_cache;

/* Block table and slot map of one step, from the requests' lengths, on the device. Request r (of rows,
 * 1...8192) holds the first ceil(lens[r] / page_size) entries of its row of table [rows][table_stride].
 *   append[r] >= 0: the step appends that many tokens to it; append[r] < 0: the request has ended.
 * Ended requests' pages go onto the end of free_list (capacity `pages` entries, the first *free_count of
 * them valid), in request order; entries outside [0, pages), of pages given up before, are no pages and are passed
 * over. The pages the appended tokens need then come off its end, in request
 * order, as long as they last: a request is refused (nothing granted, nothing appended) when the pages
 * needed up to and including it exceed the free ones, when it would outgrow its table row, or when its
 * tokens pass the `tokens` capacity. Outputs: the granted pages in table; new_lens[r] (0 for an ended
 * request, unchanged for a refused one); row_start[0..rows], the running sums of the appended counts (the
 * step's tokens are packed in request order); for each of `tokens` packed tokens its position and its slot
 * (page * page_size + offset), both -1 for a refused request's tokens and past the last token; counts[4]:
 * free pages left (the next step's free_count), tokens, pages granted, requests refused. An ended
 * request's table row is left as it was. Entries outside [0, pages) give slot -1. table and free_list are
 * updated in place; no array that is written may overlap another one. All values int32. */
PLAMO_API int plamo_k_paged_plan(const int32_t* lens, const int32_t* append, int rows, int page_size, int pages,
                                 int32_t* table, int table_stride, int32_t* free_list, const int32_t* free_count,
                                 int32_t* new_lens, int32_t* row_start, int32_t* slots, int32_t* positions, int tokens,
                                 int32_t* counts, void* stream);

/* QK-norm, rotary embedding and cache append of `tokens` rows of a q/k/v projection, as the forward's own
 * (Kernels.metal:223-274) but in fp32 with one rounding at the end: a row of qkv (qkv_stride elements
 * apart) holds heads + 2 * kv_heads heads of head_dim; query and key heads become
 *   x * rsqrt(mean(x^2) + eps) * (1 + w)   (w = q_norm / k_norm, [head_dim]; NULL: no norm)
 * and are rotated (rotate-half) by the row of rope [rope_rows][head_dim / 2] at the token's position (u32 =
 * bf16 cos bits | sin bits << 16; NULL: no rotation, positions unused). Queries go to q (q_stride elements
 * apart), keys and values to the cache's slot slots[t]. A token whose slot is outside the cache or whose
 * position is outside rope is not appended and its query row is zero. Two tokens must not share a slot; q and
 * the cache must not overlap qkv.
 * Pointers 16-byte aligned, strides multiples of 8. */
PLAMO_API int plamo_k_paged_qkv(const plamo_paged_cache* cache, const void* qkv, int64_t qkv_stride, int tokens, int heads,
                                const void* q_norm, const void* k_norm, float eps, const uint32_t* rope, int rope_rows,
                                const int32_t* positions, const int32_t* slots, void* q, int64_t q_stride, void* stream);

/* Attention of one new token of every request over its pages. Request r (of rows, 1...8192) sees the keys
 * at positions [max(0, n - window), n), n = min(lens[r], max_len) (window 0: all of them); the key at
 * position p is in page table[r][p / page_size]; entries outside [0, pages) hold no keys (a page given up
 * behind the window). max_len bounds the lengths for the launch: at most table_stride * page_size. How the work is split
 * is chosen by it, so short requests run faster under a bound near their longest.
 * row_start NULL: request r's query is row r of q [q_rows][heads][head_dim] (q_stride elements apart), and
 * q_rows >= rows. Else it is row row_start[r + 1] - 1 (the request's last packed token of
 * plamo_k_paged_plan), and requests without a token are skipped. heads: a multiple of kv_heads, at most 256.
 *   out = sum_j softmax_j(scale * q.k_j) v_j (scale > 0) in fp32 (the probabilities enter the products as hi + lo pairs
 *   of the 16-bit type), rounded once; lse (may be NULL, [q_rows][heads] fp32) = ln sum_j exp(scale * q.k_j).
 * An infinite value of a visible key makes its output that infinity, as long as the key's probability is at least 2^-126
 * of the request's largest (below, fp32 holds no probability: NaN).
 * A request that sees no key, or whose scores are all -inf, gets zeros and lse -inf. Query rows that belong
 * to no request are not written. `workspace`: 16-byte aligned device memory of at least
 * plamo_k_paged_attention_workspace() bytes, no initial contents needed; calls that share one must not
 * overlap. out, lse and workspace lie apart from each other and from every input. Pointers 16-byte aligned, strides
 * multiples of 8. */
PLAMO_API int plamo_k_paged_attention(const plamo_paged_cache* cache, const void* q, int64_t q_stride, int q_rows, int heads,
                                      const int32_t* table, int table_stride, const int32_t* lens, int rows,
                                      const int32_t* row_start, int max_len, int window, float scale, void* out,
                                      int64_t out_stride, float* lse, void* workspace, size_t workspace_bytes,
                                      void* stream);

/* Bytes of workspace that every plamo_k_paged_attention call accepts (no device needed). */
PLAMO_API size_t plamo_k_paged_attention_workspace(void);

/* Samples one id per row of logits [rows][vocab] (row_stride elements apart; dtype 0 bf16, 1 fp16, 2 fp32;
 * vocab <= 2^22) by per-row controls on the device (each array NULL: that control off for every row):
 *   temperature > 0; <= 0 or NaN: greedy (the lowest index of the largest logit). NULL: 1
 *   top_k > 0: only the top_k largest logits. top_p < 1: only the shortest run of them, in descending
 *   order, that holds at least top_p of their probability (to 2^-24; never empty). min_p > 0: only ids at
 *   least min_p times as likely as the most likely one. Ties go to the lower index.
 * A probability is a whole number w = floor(2^40 * exp((logit - max) / temperature)) (the fp32 exponential),
 * so every sum is exact and the id does not depend on how the work is split. With u[row] in [0, 1) the
 * id is the lowest kept index at which the running sum of kept w exceeds floor(2^24 u) * W / 2^24, W the
 * sum of all kept w. ids[row]; logprobs[row] (may be NULL) = ln(w_id / W); kept[row] (may be NULL) the number
 * of kept ids. NaN and -inf logits are never chosen; a row of only those gives id 0, logprob -inf and kept 0.
 * Equal +inf logits share the probability. ids, logprobs and kept lie apart from each other and from every input. */
PLAMO_API int plamo_k_sample(const void* logits, int dtype, int rows, int vocab, int64_t row_stride,
                             const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                             const float* u, int32_t* ids, float* logprobs, int32_t* kept, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* PLAMO_KERNELS_H */
