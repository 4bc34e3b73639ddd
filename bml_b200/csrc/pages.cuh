// pages.cuh -- launch interface of the kernels that share, return and move the
// pages of a paged cache, and of the verification of drafted tokens.
#pragma once

#include "paged.cuh"

namespace bml {

// launch_after for a kernel whose CTAs work in clusters of `cluster`.
template <typename... KArgs, typename... Args>
cudaError_t launch_clusters(void (*kernel)(KArgs...), uint32_t cluster, dim3 grid, int threads, int smem, cudaStream_t st,
                            const Args &...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// status bits of a fork or a release (the first two are a plan's)
constexpr int32_t kPageShared = 8;

// What a pool's kernels share: the layers' pools, whose pages are page_bytes long.
struct PoolParams {
    char *k_pool, *v_pool;  // [n_layers] pools, layer_bytes apart
    uint32_t n_layers, n_pages, page_shift;
    uint64_t layer_bytes;
    uint32_t row_bytes;
};

struct ForkParams {
    PoolParams pool;
    const int32_t *src, *dst;  // [m]
    uint32_t m;
    const int32_t *lens, *owned;  // [n]
    uint32_t n, max_pages;
    int32_t *table;               // [n][max_pages], rows dst written
    const int32_t *shared;        // [n_pages]
    const int32_t *free_pages;    // [n_free]; the first *free_used are taken
    uint32_t n_free;
    const int32_t *free_used;
    int32_t *lens_out, *owned_out, *shared_out, *free_used_out, *status;
    int num_sms;
};
cudaError_t launch_page_fork(const ForkParams &p, cudaStream_t st);

struct FreeParams {
    const int32_t *keep, *lens, *owned;  // [n]
    uint32_t n, max_pages, n_pages, page_shift;
    const int32_t *table, *shared, *free_pages;
    uint32_t n_free;
    const int32_t *free_used;
    int32_t *lens_out, *owned_out, *shared_out, *free_out, *free_used_out, *status;
    uint32_t *work;  // free_work_bytes(n_free)
    uint32_t tile;   // entries of the free list a CTA, set by the launch
    int num_sms;
};
constexpr uint32_t kFreeTiles = 1024;  // at most
constexpr uint64_t free_work_bytes(uint32_t n_free) { return 4ull * (kFreeTiles + (n_free + 31ull) / 32); }
cudaError_t launch_page_free(const FreeParams &p, cudaStream_t st);

struct CompactParams {
    PoolParams pool;
    const int32_t *owned;  // [n]
    uint32_t n, max_pages;
    const int32_t *table, *shared;
    int32_t *table_out, *shared_out, *free_out, *free_used_out;
    int32_t *work;  // [3 * n_pages + 1]
    int num_sms;
};
cudaError_t launch_page_compact(const CompactParams &p, cudaStream_t st);

struct VerifyParams {
    const void *target, *draft;  // [n_tokens][vocab]; draft null: the tokens were picked, not drawn
    const int32_t *tokens, *parents;
    const int32_t *node_start;  // [n + 1]
    uint32_t n, n_tokens, vocab;
    const float *u, *u_next;  // [n_tokens], [n]
    uint32_t max_path;
    int32_t *path, *n_accept, *next;  // [n][max_path], [n], [n]
    bml_dtype type;
    int num_sms;
};
cudaError_t launch_verify_drafts(const VerifyParams &p, cudaStream_t st);

}  // namespace bml
