// paged.cuh -- launch interface of the paged-cache kernels: page planning,
// RoPE append through slots, and the commit of an accepted path.
#pragma once

#include "common.cuh"

namespace bml {

// A launch that may begin while the kernel before it on the stream ends; the
// kernels wait for that kernel (griddepcontrol.wait) before they read or write
// global memory.
template <typename... KArgs, typename... Args>
cudaError_t launch_after(void (*kernel)(KArgs...), dim3 grid, int threads, int smem, cudaStream_t st, const Args &...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

constexpr uint32_t kPlanMaxSeqs = 4096;  // requests of one plan (their prefix sums live in shared memory)
constexpr uint32_t kTreeMaxNodes = 256;  // drafted tokens of one request (4 mask words)

// status bits of a plan
constexpr int32_t kPlanNoPages = 1, kPlanBad = 2, kPlanNoRoom = 4;

struct PlanParams {
    const int32_t *lens, *n_new, *owned;  // [n]
    uint32_t n;
    const int32_t *free_pages;  // [n_free]; the first *free_used are taken
    uint32_t n_free;
    const int32_t *free_used;  // [1]
    uint32_t page_shift, max_pages;
    int32_t *table;          // [n][max_pages], new entries written
    const int32_t *parents;  // [n_tokens] or null
    uint32_t n_tokens, n_words;
    int32_t *node_start;  // [n+1]
    int32_t *kv_lens, *owned_out, *free_used_out;
    int64_t *slots;
    int32_t *positions;
    uint64_t *mask;  // [n_tokens][n_words], null without parents
    int32_t *status;
    int num_sms;
};
cudaError_t launch_page_plan(const PlanParams &p, cudaStream_t st);

struct PagedAppendParams {
    const void *q;  // null: no queries
    void *q_out;
    const void *k, *v;
    const int64_t *slots;
    const int32_t *positions;  // null: no rotation
    uint32_t n_tokens, n_heads, n_kv, d;
    double log2_theta;
    void *k_pool, *v_pool;
    uint64_t n_rows;  // rows of a pool
    bml_dtype src, dst;
    int num_sms;
};
cudaError_t launch_paged_append(const PagedAppendParams &p, cudaStream_t st);

struct CommitParams {
    char *k_pool, *v_pool;  // [n_layers] pools, layer_bytes apart
    uint32_t n_layers, n_pages, page_shift, max_pages;
    uint64_t layer_bytes;
    uint32_t row_bytes;
    const int32_t *table, *lens, *kv_lens, *node_start;
    uint32_t n;
    const int32_t *path;  // [n][max_path]
    uint32_t max_path;
    const int32_t *n_accept;
    int32_t *lens_out;
};
cudaError_t launch_paged_commit(const CommitParams &p, cudaStream_t st);

}  // namespace bml
