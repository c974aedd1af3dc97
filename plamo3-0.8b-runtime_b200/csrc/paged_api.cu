// Kernel-level C ABI of the paged serving step (include/plamo_kernels.h): argument checks and launches.
#include "../../include/plamo_kernels.h"
#include "paged.h"

#include <climits>
#include <cmath>
#include <cstdio>
#include <initializer_list>
#include <string>

namespace plamo {
extern thread_local std::string g_error;
}
using namespace plamo;

namespace {

// Nothing may be thrown through the C entry points: without memory for its words a failure stays a status.
int invalid(const char* what, const char* more = "") {
    try {
        g_error = std::string(what) + more;
    } catch (...) {
    }
    return 1;
}
int launched(cudaError_t e) { return e == cudaSuccess ? 0 : invalid("CUDA error: ", cudaGetErrorString(e)); }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// Whether arrays of 32-bit values (null ones aside) lie on 4-byte boundaries.
bool aligned4(std::initializer_list<const void*> arrays) {
    for (const void* p : arrays)
        if (reinterpret_cast<uintptr_t>(p) & 3) return false;
    return true;
}
constexpr const char* MISALIGNED = "Arrays of 32-bit values must be 4-byte aligned";

// The bytes of an array of n 32-bit values.
struct Range {
    uintptr_t begin, end;
};
Range range(const int32_t* p, long long n) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    return {at, at + uintptr_t(n) * 4};
}
bool overlap(const Range& x, const Range& y) { return x.begin < y.end && y.begin < x.end; }

// Null, or the words that say what is wrong with a cache descriptor.
const char* cache_fault(const plamo_paged_cache* c) {
    if (!c || !c->keys || !c->values) return "Invalid paged cache";
    if (c->dtype != 0 && c->dtype != 1) return "A paged cache is bf16 (0) or fp16 (1)";
    if (c->head_dim != 64 && c->head_dim != 128) return "A paged cache's head_dim is 64 or 128";
    if (c->pages < 1 || c->page_size < 1 || c->kv_heads < 1 || c->kv_heads > 256 ||
        (long long)c->pages * c->page_size > INT_MAX)
        return "Invalid paged cache geometry";
    if (!aligned16(c->keys) || !aligned16(c->values) || c->page_stride % 8 || c->token_stride % 8 || c->head_stride % 8 ||
        c->page_stride < 0 || c->token_stride < 0 || c->head_stride < 0)
        return "A paged cache needs 16-byte aligned tensors and strides that are multiples of 8";
    return nullptr;
}
PagedCacheArgs cache_args(const plamo_paged_cache* c) {
    return PagedCacheArgs{static_cast<uint16_t*>(c->keys), static_cast<uint16_t*>(c->values), c->pages, c->page_size,
                          c->kv_heads, c->page_stride, c->token_stride, c->head_stride};
}

}  // namespace

extern "C" {

int plamo_k_paged_plan(const int32_t* lens, const int32_t* append, int rows, int page_size, int pages, int32_t* table,
                       int table_stride, int32_t* free_list, const int32_t* free_count, int32_t* new_lens,
                       int32_t* row_start, int32_t* slots, int32_t* positions, int tokens, int32_t* counts, void* stream) {
    if (!lens || !append || !table || !free_list || !free_count || !new_lens || !row_start || !slots || !positions ||
        !counts || rows < 1 || rows > PAGED_MAX_ROWS || page_size < 1 || pages < 1 || table_stride < 1 || tokens < 1 ||
        tokens > INT_MAX - 64 * PAGED_MAX_ROWS || (long long)pages * page_size > INT_MAX ||
        (long long)rows * table_stride > INT_MAX)
        return invalid("Invalid paged plan arguments");
    if (!aligned4({lens, append, table, free_list, free_count, new_lens, row_start, slots, positions, counts}))
        return invalid(MISALIGNED);
    // every array that is written, table and free_list among them, lies apart from every other one
    const Range written[] = {range(table, (long long)rows * table_stride), range(free_list, pages), range(new_lens, rows),
                             range(row_start, rows + 1ll), range(slots, tokens), range(positions, tokens), range(counts, 4)};
    const Range read[] = {range(lens, rows), range(append, rows), range(free_count, 1)};
    for (const Range& w : written) {
        for (const Range& r : read)
            if (overlap(w, r)) return invalid("A paged plan's outputs must not overlap its inputs");
        for (const Range& o : written)
            if (&o != &w && overlap(w, o)) return invalid("A paged plan's outputs must not overlap each other");
    }
    return launched(launch_paged_plan({lens, append, rows, page_size, pages, table, table_stride, free_list, free_count,
                                       new_lens, row_start, slots, positions, tokens, counts},
                                      static_cast<cudaStream_t>(stream)));
}

int plamo_k_paged_qkv(const plamo_paged_cache* cache, const void* qkv, int64_t qkv_stride, int tokens, int heads,
                      const void* q_norm, const void* k_norm, float eps, const uint32_t* rope, int rope_rows,
                      const int32_t* positions, const int32_t* slots, void* q, int64_t q_stride, void* stream) {
    if (const char* fault = cache_fault(cache)) return invalid(fault);
    const long long width = ((long long)heads + 2ll * cache->kv_heads) * cache->head_dim;
    if (!qkv || !slots || !q || tokens < 1 || heads < 1 || heads > 256 || qkv_stride < width || qkv_stride % 8 ||
        q_stride < (long long)heads * cache->head_dim || q_stride % 8 || (rope && (rope_rows < 1 || !positions)) ||
        !(eps >= 0.f))
        return invalid("Invalid paged qkv arguments");
    if ((long long)tokens * (heads + 2 * cache->kv_heads) > INT_MAX / 2) return invalid("Too many tokens in one paged qkv call");
    if (!aligned4({positions, slots})) return invalid(MISALIGNED);
    if (!aligned16(qkv) || !aligned16(q_norm) || !aligned16(k_norm) || !aligned16(rope) || !aligned16(q))
        return invalid("Paged qkv pointers must be 16-byte aligned");
    return launched(launch_paged_qkv({cache_args(cache), static_cast<const uint16_t*>(qkv), qkv_stride, tokens, heads,
                                      static_cast<const uint16_t*>(q_norm), static_cast<const uint16_t*>(k_norm), eps, rope,
                                      rope_rows, positions, slots, static_cast<uint16_t*>(q), q_stride},
                                     cache->head_dim, cache->dtype == 1, static_cast<cudaStream_t>(stream)));
}

size_t plamo_k_paged_attention_workspace(void) { return paged_attention_workspace(); }

int plamo_k_paged_attention(const plamo_paged_cache* cache, const void* q, int64_t q_stride, int q_rows, int heads,
                            const int32_t* table, int table_stride, const int32_t* lens, int rows, const int32_t* row_start,
                            int max_len, int window, float scale, void* out, int64_t out_stride, float* lse,
                            void* workspace, size_t workspace_bytes, void* stream) {
    if (const char* fault = cache_fault(cache)) return invalid(fault);
    if (!q || !table || !lens || !out || rows < 1 || rows > PAGED_MAX_ROWS || q_rows < 1 || (!row_start && q_rows < rows) ||
        heads < 1 || heads > 256 || heads % cache->kv_heads || table_stride < 1 || max_len < 1 || max_len > (1 << 30) ||
        max_len > (long long)table_stride * cache->page_size || window < 0 || !std::isfinite(scale) || !(scale > 0.f) ||
        q_stride < (long long)heads * cache->head_dim || out_stride < (long long)heads * cache->head_dim || q_stride % 8 ||
        out_stride % 8)
        return invalid("Invalid paged attention arguments");
    if (!aligned4({table, lens, row_start, lse})) return invalid(MISALIGNED);
    if (!aligned16(q) || !aligned16(out)) return invalid("Paged attention pointers must be 16-byte aligned");
    if (!workspace || !aligned16(workspace) || workspace_bytes < paged_attention_workspace()) {
        char words[96];
        std::snprintf(words, sizeof words, "Paged attention workspace too small or not 16-byte aligned: %zu bytes needed",
                      paged_attention_workspace());
        return invalid(words);
    }
    PagedAttnArgs a{cache_args(cache), static_cast<const uint16_t*>(q), q_stride, q_rows, heads, table, table_stride, lens,
                    rows, row_start, max_len, window, float(double(scale) * 1.4426950408889634), static_cast<uint16_t*>(out),
                    out_stride, lse, workspace};
    return launched(launch_paged_attention(a, cache->head_dim, cache->dtype == 1, static_cast<cudaStream_t>(stream)));
}

int plamo_k_sample(const void* logits, int dtype, int rows, int vocab, int64_t row_stride, const float* temperature,
                   const int32_t* top_k, const float* top_p, const float* min_p, const float* u, int32_t* ids,
                   float* logprobs, int32_t* kept, void* stream) {
    if (!logits || !u || !ids || dtype < 0 || dtype > 2 || rows < 1 || rows > 65535 || vocab < 1 ||
        vocab > SAMPLE_MAX_VOCAB || row_stride < vocab || (reinterpret_cast<uintptr_t>(logits) & (dtype == 2 ? 3 : 1)))
        return invalid("Invalid sample arguments");
    if (!aligned4({temperature, top_k, top_p, min_p, u, ids, logprobs, kept})) return invalid(MISALIGNED);
    return launched(launch_sample({logits, rows, vocab, row_stride, temperature, top_k, top_p, min_p, u, ids, logprobs, kept},
                                  dtype, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
