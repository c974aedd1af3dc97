// Internal interfaces of the paged serving step: argument blocks and launchers of paged_plan.cu,
// paged_qkv.cu, paged_attn.cu and sample.cu. The public contract is in include/plamo_kernels.h; every
// launcher expects arguments that paged_api.cu has checked.
#pragma once
#include <atomic>
#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace plamo {

constexpr int PAGED_MAX_ROWS = 8192;     // rows of a plan or an attention call: their prefix sums sit in shared memory
constexpr int SAMPLE_MAX_VOCAB = 1 << 22;  // 2^22 weights of at most 2^40: sums below 2^62

// Opts a kernel into `bytes` of dynamic shared memory, once a device (`done` remembers which).
template <typename Kernel>
cudaError_t allow_shared(Kernel kernel, size_t bytes, std::atomic<uint64_t>& done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || (dev < 64 && (done.load() >> dev & 1))) return e;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes));
    if (e == cudaSuccess && dev < 64) done.fetch_or(1ull << dev);
    return e;
}

struct PagedCacheArgs {
    uint16_t* keys;
    uint16_t* values;
    int pages, page_size, kv_heads;
    long long page_stride, token_stride, head_stride;
};

struct PagedPlanArgs {
    const int* lens;
    const int* append;
    int rows, page_size, pages;
    int* table;
    int table_stride;
    int* free_list;
    const int* free_count;
    int* new_lens;
    int* row_start;
    int* slots;
    int* positions;
    int tokens;
    int* counts;
};
cudaError_t launch_paged_plan(const PagedPlanArgs& a, cudaStream_t s);

struct PagedQkvArgs {
    PagedCacheArgs cache;
    const uint16_t* qkv;
    long long qkv_stride;
    int tokens, heads;
    const uint16_t* q_norm;
    const uint16_t* k_norm;
    float eps;
    const uint32_t* rope;
    int rope_rows;
    const int* positions;
    const int* slots;
    uint16_t* q;
    long long q_stride;
};
cudaError_t launch_paged_qkv(const PagedQkvArgs& a, int head_dim, bool half, cudaStream_t s);

struct PagedAttnArgs {
    PagedCacheArgs cache;
    const uint16_t* q;
    long long q_stride;
    int q_rows, heads;
    const int* table;
    int table_stride;
    const int* lens;
    int rows;
    const int* row_start;
    int max_len, window;
    float scale_log2;  // scale * log2 e: scores are kept in powers of two
    uint16_t* out;
    long long out_stride;
    float* lse;
    void* workspace;
};
size_t paged_attention_workspace();
cudaError_t launch_paged_attention(const PagedAttnArgs& a, int head_dim, bool half, cudaStream_t s);

struct SampleArgs {
    const void* logits;
    int rows, vocab;
    long long row_stride;
    const float* temperature;
    const int* top_k;
    const float* top_p;
    const float* min_p;
    const float* u;
    int* ids;
    float* logprobs;
    int* kept;
};
cudaError_t launch_sample(const SampleArgs& a, int dtype, cudaStream_t s);

}  // namespace plamo
