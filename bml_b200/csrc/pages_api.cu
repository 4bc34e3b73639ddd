// pages_api.cu -- C entry points of the pages' kernels and of the verification of
// drafted tokens (include/bml_attn.h).  Arguments are checked on the host before
// anything is launched; what lives on the device is bounded by the kernels.
#include "paged_check.cuh"
#include "pages.cuh"

namespace {

bml_status count(const char *fn, const char *what, uint32_t n) {
    if (n == 0 || n > bml::kPlanMaxSeqs) return api_fail(BML_E_INVALID, "%s: %u %s (1 to %u)", fn, n, what, bml::kPlanMaxSeqs);
    return BML_OK;
}

// The pools of a call that moves pages.
bml_status pools(const char *fn, void *k_pool, void *v_pool, uint32_t n_layers, uint32_t n_pages, uint32_t page_size, uint32_t n_kv,
                 uint32_t d, bml_dtype type, bml::PoolParams &p, uint64_t &bytes) {
    if (!valid_dtype(type)) return api_fail(BML_E_INVALID, "%s: unknown dtype", fn);
    if (n_layers == 0 || n_layers > 32767 || n_pages == 0 || n_kv == 0 || d == 0)
        return api_fail(BML_E_INVALID, "%s: zero dimension or more than 32767 layers", fn);
    if ((uint64_t)n_pages * page_size >= (1ull << 31)) return api_fail(BML_E_INVALID, "%s: %u pages of %u positions", fn, n_pages, page_size);
    const uint64_t row = (uint64_t)n_kv * d, most = (1ull << 31) / page_size / bml::dtype_size(type);
    if (row >= most) return api_fail(BML_E_INVALID, "%s: a page of 2^31 bytes or more", fn);
    if (!k_pool || !v_pool || !aligned(k_pool, 4) || !aligned(v_pool, 4)) return api_fail(BML_E_INVALID, "%s: null or misaligned pool", fn);
    p.k_pool = static_cast<char *>(k_pool);
    p.v_pool = static_cast<char *>(v_pool);
    p.n_layers = n_layers;
    p.n_pages = n_pages;
    p.page_shift = (uint32_t)page_shift(page_size);
    p.row_bytes = (uint32_t)(row * bml::dtype_size(type));
    p.layer_bytes = (uint64_t)n_pages * page_size * p.row_bytes;
    bytes = p.layer_bytes * n_layers;
    return BML_OK;
}

bml_status done(cudaError_t e, const char *fn) { return e == cudaSuccess ? bml::api_ok() : bml::api_cuda_fail(e, fn); }

}  // namespace

BML_API bml_status bml_page_fork(void *k_pool, void *v_pool, uint32_t n_layers, uint32_t n_pages, uint32_t page_size,
                                 uint32_t n_kv_heads, uint32_t head_dim, bml_dtype kv_dtype, const int32_t *src,
                                 const int32_t *dst, uint32_t m, const int32_t *lens, const int32_t *owned, uint32_t n,
                                 int32_t *block_table, uint32_t max_pages, const int32_t *shared, const int32_t *free_pages,
                                 uint32_t n_free, const int32_t *free_used, int32_t *lens_out, int32_t *owned_out,
                                 int32_t *shared_out, int32_t *free_used_out, int32_t *status, void *stream) {
    const char *fn = "bml_page_fork";
    if (bml_status st = count(fn, "requests", n)) return st;
    if (m > bml::kPlanMaxSeqs) return api_fail(BML_E_INVALID, "%s: %u forks (at most %u)", fn, m, bml::kPlanMaxSeqs);
    if (bml_status st = check_pages(page_size, max_pages, fn)) return st;
    bml::ForkParams p = {};
    uint64_t pool = 0;
    if (bml_status st = pools(fn, k_pool, v_pool, n_layers, n_pages, page_size, n_kv_heads, head_dim, kv_dtype, p.pool, pool)) return st;
    if (bml_status st = ints(fn, {lens, owned, block_table, shared, free_used, lens_out, owned_out, shared_out, free_used_out})) return st;
    if (m)
        if (bml_status st = ints(fn, {src, dst, status})) return st;
    if (n_free > 0x7fffffffu) return api_fail(BML_E_INVALID, "%s: count above 2^31 - 1", fn);
    if (n_free && (!free_pages || !aligned(free_pages, 4))) return api_fail(BML_E_INVALID, "%s: null or misaligned free_pages", fn);
    const uint64_t n4 = 4ull * n, m4 = 4ull * m;
    const std::initializer_list<Span> written = {{k_pool, pool}, {v_pool, pool}, {block_table, n4 * max_pages}, {lens_out, n4}, {owned_out, n4},
                                                 {shared_out, 4ull * n_pages}, {free_used_out, 4}, {m ? status : nullptr, m4}};
    if (overlap(written, {{lens, n4}, {owned, n4}, {shared, 4ull * n_pages}, {free_pages, 4ull * n_free}, {free_used, 4},
                          {m ? src : nullptr, m4}, {m ? dst : nullptr, m4}}) ||
        overlap(written))
        return api_fail(BML_E_INVALID, "%s: the pools and results must not overlap one another or what is read", fn);
    p.src = src;
    p.dst = dst;
    p.m = m;
    p.lens = lens;
    p.owned = owned;
    p.n = n;
    p.max_pages = max_pages;
    p.table = block_table;
    p.shared = shared;
    p.free_pages = free_pages;
    p.n_free = n_free;
    p.free_used = free_used;
    p.lens_out = lens_out;
    p.owned_out = owned_out;
    p.shared_out = shared_out;
    p.free_used_out = free_used_out;
    p.status = status;
    p.num_sms = sm_count(this_device());
    return done(bml::launch_page_fork(p, static_cast<cudaStream_t>(stream)), fn);
}

BML_API bml_status bml_page_free(const int32_t *keep, const int32_t *lens, const int32_t *owned, uint32_t n,
                                 const int32_t *block_table, uint32_t max_pages, uint32_t page_size, const int32_t *shared,
                                 uint32_t n_pages, const int32_t *free_pages, uint32_t n_free, const int32_t *free_used,
                                 int32_t *lens_out, int32_t *owned_out, int32_t *shared_out, int32_t *free_out,
                                 int32_t *free_used_out, int32_t *status, void *workspace, size_t workspace_bytes,
                                 void *stream) {
    const char *fn = "bml_page_free";
    if (bml_status st = count(fn, "requests", n)) return st;
    if (bml_status st = check_pages(page_size, max_pages, fn)) return st;
    if (n_pages == 0 || (uint64_t)n_pages * page_size >= (1ull << 31))
        return api_fail(BML_E_INVALID, "%s: %u pages of %u positions", fn, n_pages, page_size);
    if (bml_status st = ints(fn, {keep, lens, owned, block_table, shared, free_used, lens_out, owned_out, shared_out, free_used_out, status,
                              static_cast<const int32_t *>(workspace)}))
        return st;
    if (n_free > 0x7fffffffu) return api_fail(BML_E_INVALID, "%s: count above 2^31 - 1", fn);
    const uint64_t need = bml::free_work_bytes(n_free);
    if (workspace_bytes < need) return api_fail(BML_E_INVALID, "%s: workspace of %zu bytes, need %llu", fn, workspace_bytes, (unsigned long long)need);
    if (n_free)
        if (bml_status st = ints(fn, {free_pages, free_out})) return st;
    const uint64_t n4 = 4ull * n, p4 = 4ull * n_pages, f4 = 4ull * n_free;
    const std::initializer_list<Span> written = {{lens_out, n4}, {owned_out, n4}, {shared_out, p4}, {n_free ? free_out : nullptr, f4},
                                                 {free_used_out, 4}, {status, n4}, {workspace, need}};
    if (overlap(written, {{keep, n4}, {lens, n4}, {owned, n4}, {block_table, n4 * max_pages}, {shared, p4}, {n_free ? free_pages : nullptr, f4},
                          {free_used, 4}}) ||
        overlap(written))
        return api_fail(BML_E_INVALID, "%s: results and workspace must not overlap one another or what is read", fn);
    bml::FreeParams p = {};
    p.keep = keep;
    p.lens = lens;
    p.owned = owned;
    p.n = n;
    p.max_pages = max_pages;
    p.n_pages = n_pages;
    p.page_shift = (uint32_t)page_shift(page_size);
    p.table = block_table;
    p.shared = shared;
    p.free_pages = free_pages;
    p.n_free = n_free;
    p.free_used = free_used;
    p.lens_out = lens_out;
    p.owned_out = owned_out;
    p.shared_out = shared_out;
    p.free_out = free_out;
    p.free_used_out = free_used_out;
    p.status = status;
    p.work = static_cast<uint32_t *>(workspace);
    p.num_sms = sm_count(this_device());
    return done(bml::launch_page_free(p, static_cast<cudaStream_t>(stream)), fn);
}

BML_API bml_status bml_page_compact(void *k_pool, void *v_pool, uint32_t n_layers, uint32_t n_pages, uint32_t page_size,
                                    uint32_t n_kv_heads, uint32_t head_dim, bml_dtype kv_dtype, const int32_t *owned, uint32_t n,
                                    const int32_t *block_table, uint32_t max_pages, const int32_t *shared, int32_t *table_out,
                                    int32_t *shared_out, int32_t *free_out, int32_t *free_used_out, void *workspace,
                                    size_t workspace_bytes, void *stream) {
    const char *fn = "bml_page_compact";
    if (bml_status st = count(fn, "requests", n)) return st;
    if (bml_status st = check_pages(page_size, max_pages, fn)) return st;
    bml::CompactParams p = {};
    uint64_t pool = 0;
    if (bml_status st = pools(fn, k_pool, v_pool, n_layers, n_pages, page_size, n_kv_heads, head_dim, kv_dtype, p.pool, pool)) return st;
    if (bml_status st = ints(fn, {owned, block_table, shared, table_out, shared_out, free_out, free_used_out, static_cast<const int32_t *>(workspace)}))
        return st;
    const uint64_t n4 = 4ull * n, p4 = 4ull * n_pages, need = 3 * p4 + 4;
    if (workspace_bytes < need) return api_fail(BML_E_INVALID, "%s: workspace of %zu bytes, need %llu", fn, workspace_bytes, (unsigned long long)need);
    const std::initializer_list<Span> written = {{k_pool, pool}, {v_pool, pool}, {table_out, n4 * max_pages}, {shared_out, p4}, {free_out, p4},
                                                 {free_used_out, 4}, {workspace, need}};
    if (overlap(written, {{owned, n4}, {block_table, n4 * max_pages}, {shared, p4}}) || overlap(written))
        return api_fail(BML_E_INVALID, "%s: the pools, results and workspace must not overlap one another or what is read", fn);
    p.owned = owned;
    p.n = n;
    p.max_pages = max_pages;
    p.table = block_table;
    p.shared = shared;
    p.table_out = table_out;
    p.shared_out = shared_out;
    p.free_out = free_out;
    p.free_used_out = free_used_out;
    p.work = static_cast<int32_t *>(workspace);
    p.num_sms = sm_count(this_device());
    return done(bml::launch_page_compact(p, static_cast<cudaStream_t>(stream)), fn);
}

BML_API bml_status bml_verify_drafts(const void *target, const void *draft, bml_dtype dtype, uint32_t vocab, const int32_t *tokens,
                                     const int32_t *parents, uint32_t n_tokens, const int32_t *node_start, uint32_t n,
                                     const float *u, const float *u_next, uint32_t max_path, int32_t *path, int32_t *n_accept,
                                     int32_t *next, void *stream) {
    const char *fn = "bml_verify_drafts";
    if (!valid_dtype(dtype)) return api_fail(BML_E_INVALID, "%s: unknown dtype", fn);
    if (n == 0 || n > 0x7fffffu) return api_fail(BML_E_INVALID, "%s: %u requests (1 to 2^23 - 1)", fn, n);
    if (vocab == 0 || vocab > 0x7fffffffu || n_tokens > 0x7fffffffu || max_path == 0 || max_path > 0x7fffffffu)
        return api_fail(BML_E_INVALID, "%s: vocab, n_tokens or max_path is zero or above 2^31 - 1", fn);
    if (bml_status st = ints(fn, {node_start, path, n_accept, next, reinterpret_cast<const int32_t *>(u_next)})) return st;
    if (n_tokens) {
        if (bml_status st = ints(fn, {tokens, parents, reinterpret_cast<const int32_t *>(u)})) return st;
        if (!target || !aligned(target, bml::dtype_size(dtype)) || !aligned(draft, bml::dtype_size(dtype)))
            return api_fail(BML_E_INVALID, "%s: null or misaligned probabilities", fn);
    }
    const uint64_t n4 = 4ull * n, t4 = n_tokens ? 4ull * n_tokens : 0, rows = (uint64_t)n_tokens * vocab * bml::dtype_size(dtype);
    const std::initializer_list<Span> written = {{path, n4 * max_path}, {n_accept, n4}, {next, n4}};
    auto some = [&](const void *x) { return n_tokens ? x : nullptr; };
    if (overlap(written, {{some(target), rows}, {some(draft), rows}, {some(tokens), t4}, {some(parents), t4}, {some(u), t4}, {u_next, n4},
                          {node_start, n4 + 4}}) ||
        overlap(written))
        return api_fail(BML_E_INVALID, "%s: results must not overlap one another or what is read", fn);
    bml::VerifyParams p = {};
    p.target = target;
    p.draft = draft;
    p.tokens = tokens;
    p.parents = parents;
    p.node_start = node_start;
    p.n = n;
    p.n_tokens = n_tokens;
    p.vocab = vocab;
    p.u = u;
    p.u_next = u_next;
    p.max_path = max_path;
    p.path = path;
    p.n_accept = n_accept;
    p.next = next;
    p.type = dtype;
    p.num_sms = sm_count(this_device());
    return done(bml::launch_verify_drafts(p, static_cast<cudaStream_t>(stream)), fn);
}
