// paged_api.cu -- C entry points of the paged cache and of the attention of
// drafted tokens (include/bml_attn.h).  Arguments are checked on the host
// before anything is launched; sizes that live on the device are bounded by
// the kernels themselves.
#include <math.h>

#include "../../include/bml_diag.h"
#include "paged_check.cuh"
#include "tree.cuh"

BML_API bml_status bml_paged_plan(const int32_t *lens, const int32_t *n_new, const int32_t *owned, uint32_t n,
                                  const int32_t *free_pages, uint32_t n_free, const int32_t *free_used,
                                  uint32_t page_size, uint32_t max_pages, int32_t *block_table,
                                  const int32_t *parents, uint32_t n_tokens, uint32_t n_words, int32_t *node_start,
                                  int32_t *kv_lens, int32_t *owned_out, int32_t *free_used_out, int64_t *slots,
                                  int32_t *positions, uint64_t *mask, int32_t *status, void *stream) {
    const char *fn = "bml_paged_plan";
    if (n == 0 || n > bml::kPlanMaxSeqs) return api_fail(BML_E_INVALID, "%s: %u requests (1 to %u)", fn, n, bml::kPlanMaxSeqs);
    if (bml_status st = check_pages(page_size, max_pages, fn)) return st;
    if (bml_status st = ints(fn, {lens, n_new, owned, free_used, block_table, node_start, kv_lens, owned_out, free_used_out, status}))
        return st;
    if (n_free > 0x7fffffffu || n_tokens > 0x7fffffffu) return api_fail(BML_E_INVALID, "%s: count above 2^31 - 1", fn);
    if (n_free && (!free_pages || !aligned(free_pages, 4))) return api_fail(BML_E_INVALID, "%s: null or misaligned free_pages", fn);
    if (n_tokens && (!slots || !aligned(slots, 8) || !positions || !aligned(positions, 4)))
        return api_fail(BML_E_INVALID, "%s: null or misaligned slots or positions", fn);
    if (n_tokens && parents) {
        if (n_words < 1 || n_words > bml::kTreeMaxNodes / 64) return api_fail(BML_E_INVALID, "%s: %u mask words (1 to 4)", fn, n_words);
        if (!aligned(parents, 4) || !mask || !aligned(mask, 8))
            return api_fail(BML_E_INVALID, "%s: parents need a mask (both aligned)", fn);
    }
    const uint64_t n4 = 4ull * n, t4 = 4ull * n_tokens;
    const bool drafts = n_tokens && parents;
    const std::initializer_list<Span> written = {{node_start, n4 + 4}, {kv_lens, n4}, {owned_out, n4}, {free_used_out, 4}, {status, n4},
                                                 {slots, 2 * t4}, {positions, t4}, {drafts ? mask : nullptr, 2 * t4 * n_words},
                                                 {block_table, n4 * max_pages}};
    if (overlap(written, {{lens, n4}, {n_new, n4}, {owned, n4}, {free_pages, 4ull * n_free}, {free_used, 4}, {drafts ? parents : nullptr, t4}}))
        return api_fail(BML_E_INVALID, "%s: results need buffers of their own, not those of lens, n_new, owned, parents or the free list", fn);
    if (overlap(written)) return api_fail(BML_E_INVALID, "%s: results overlap one another", fn);
    bml::PlanParams p = {};
    p.lens = lens;
    p.n_new = n_new;
    p.owned = owned;
    p.n = n;
    p.free_pages = free_pages;
    p.n_free = n_free;
    p.free_used = free_used;
    p.page_shift = (uint32_t)page_shift(page_size);
    p.max_pages = max_pages;
    p.table = block_table;
    p.parents = n_tokens ? parents : nullptr;
    p.n_tokens = n_tokens;
    p.n_words = n_words;
    p.node_start = node_start;
    p.kv_lens = kv_lens;
    p.owned_out = owned_out;
    p.free_used_out = free_used_out;
    p.slots = slots;
    p.positions = positions;
    p.mask = p.parents ? mask : nullptr;
    p.status = status;
    p.num_sms = sm_count(this_device());
    const cudaError_t e = bml::launch_page_plan(p, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? bml::api_ok() : bml::api_cuda_fail(e, fn);
}

BML_API bml_status bml_paged_append(const void *q_dev, const void *k_dev, const void *v_dev, bml_dtype src_dtype,
                                    const int64_t *slots, const int32_t *positions, uint32_t n_tokens,
                                    uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim, double theta,
                                    void *q_out_dev, void *k_pool, void *v_pool, bml_dtype kv_dtype, uint64_t n_rows,
                                    void *stream) {
    const char *fn = "bml_paged_append";
    if (!valid_dtype(src_dtype) || !valid_dtype(kv_dtype)) return api_fail(BML_E_INVALID, "%s: unknown dtype", fn);
    if (n_kv_heads == 0 || head_dim == 0) return api_fail(BML_E_INVALID, "%s: zero dimension", fn);
    if (head_dim % 2) return api_fail(BML_E_INVALID, "%s: head_dim %u is odd", fn, head_dim);
    if (head_dim > 1024 || n_kv_heads > 65536 || n_heads > 65536) return api_fail(BML_E_UNSUPPORTED, "%s: head_dim %u (at most 1024) or head count", fn, head_dim);
    if ((q_dev == nullptr) != (q_out_dev == nullptr)) return api_fail(BML_E_INVALID, "%s: q and q_out come together", fn);
    if (q_dev && n_heads == 0) return api_fail(BML_E_INVALID, "%s: zero q heads", fn);
    if (positions && !(theta > 0.0 && isfinite(theta))) return api_fail(BML_E_INVALID, "%s: theta must be positive", fn);
    if (positions && theta < 1.0 / 65536) return api_fail(BML_E_UNSUPPORTED, "%s: theta %g (at least 2^-16)", fn, theta);
    if (n_tokens == 0) return bml::api_ok();
    if (n_tokens > 0x7fffffffu || n_rows > 0x7fffffffull) return api_fail(BML_E_INVALID, "%s: count above 2^31 - 1", fn);
    if (!k_dev || !v_dev || !k_pool || !v_pool || !slots) return api_fail(BML_E_INVALID, "%s: null pointer", fn);
    const size_t es = 2 * bml::dtype_size(src_dtype), ed = 2 * bml::dtype_size(kv_dtype);
    if (!aligned(q_dev, es) || !aligned(q_out_dev, es) || !aligned(k_dev, es) || !aligned(v_dev, es) || !aligned(k_pool, ed) ||
        !aligned(v_pool, ed) || !aligned(slots, 8) || !aligned(positions, 4))
        return api_fail(BML_E_INVALID, "%s: misaligned pointer", fn);
    if (q_dev != q_out_dev) {
        const uintptr_t a = reinterpret_cast<uintptr_t>(q_dev), b = reinterpret_cast<uintptr_t>(q_out_dev);
        const uint64_t bytes = (uint64_t)n_tokens * n_heads * head_dim * bml::dtype_size(src_dtype);
        if ((a < b ? b - a : a - b) < bytes) return api_fail(BML_E_INVALID, "%s: q_out overlaps q", fn);
    }
    // tokens are read and stored by CTAs of their own
    const uint64_t row = (uint64_t)n_kv_heads * head_dim, src = (uint64_t)n_tokens * row * bml::dtype_size(src_dtype);
    const uint64_t qb = (uint64_t)n_tokens * n_heads * head_dim * bml::dtype_size(src_dtype), pool = n_rows * row * bml::dtype_size(kv_dtype);
    if (overlap({{k_pool, pool}, {v_pool, pool}, {q_out_dev, qb}},
                {{k_dev, src}, {v_dev, src}, {slots, 8ull * n_tokens}, {positions, 4ull * n_tokens}}) ||
        overlap({{k_pool, pool}, {v_pool, pool}}, {{q_dev, qb}}) || overlap({{k_pool, pool}, {v_pool, pool}, {q_out_dev, qb}}))
        return api_fail(BML_E_INVALID, "%s: the pools and q_out must not overlap one another or what is read", fn);
    bml::PagedAppendParams p = {};
    p.q = q_dev;
    p.q_out = q_out_dev;
    p.k = k_dev;
    p.v = v_dev;
    p.slots = slots;
    p.positions = positions;
    p.n_tokens = n_tokens;
    p.n_heads = q_dev ? n_heads : 0;
    p.n_kv = n_kv_heads;
    p.d = head_dim;
    p.log2_theta = log2(theta);
    p.k_pool = k_pool;
    p.v_pool = v_pool;
    p.n_rows = n_rows;
    p.src = src_dtype;
    p.dst = kv_dtype;
    p.num_sms = sm_count(this_device());
    const cudaError_t e = bml::launch_paged_append(p, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? bml::api_ok() : bml::api_cuda_fail(e, fn);
}

BML_API bml_status bml_attn_tree_workspace_size(uint32_t head_dim, int32_t device, size_t *bytes) {
    const char *fn = "bml_attn_tree_workspace_size";
    if (!bytes) return api_fail(BML_E_INVALID, "%s: null pointer", fn);
    if (head_dim != 64 && head_dim != 128) return api_fail(BML_E_UNSUPPORTED, "%s: head_dim %u (supported: 64, 128)", fn, head_dim);
    *bytes = bml::tree_workspace_bytes(head_dim, sm_count(device));
    return bml::api_ok();
}

namespace {

// What bml_attn_tree_sized takes, and what only tests set.  chunk: bml_attn_chunk.
bml_status attn_tree(const char *fn, bool chunk, const void *q_dev, bml_dtype q_dtype, uint32_t n_tokens, uint32_t n_heads,
                     uint32_t n_kv_heads, uint32_t head_dim, const void *k_pool, const void *v_pool, bml_dtype kv_dtype,
                     uint32_t n_pages, uint32_t page_size, const int32_t *block_table, uint32_t max_pages,
                     const int32_t *kv_lens, const int32_t *node_start, uint32_t n_seqs, const uint64_t *mask,
                     uint32_t n_words, float scale, void *out_dev, void *workspace, size_t workspace_bytes,
                     uint32_t n_live, uint32_t max_nodes, uint64_t wait_ns, uint32_t diag, void *stream) {
    if (!valid_dtype(q_dtype) || !valid_dtype(kv_dtype)) return api_fail(BML_E_INVALID, "%s: unknown dtype", fn);
    if (q_dtype != BML_F32 && q_dtype != kv_dtype)
        return api_fail(BML_E_UNSUPPORTED, "%s: 16-bit queries need pages of their own type", fn);
    if (n_heads == 0 || n_kv_heads == 0 || n_seqs == 0 || n_pages == 0) return api_fail(BML_E_INVALID, "%s: zero dimension", fn);
    if (n_heads % n_kv_heads) return api_fail(BML_E_INVALID, "%s: n_heads %u is not a multiple of n_kv_heads %u", fn, n_heads, n_kv_heads);
    if (head_dim != 64 && head_dim != 128) return api_fail(BML_E_UNSUPPORTED, "%s: head_dim %u (supported: 64, 128)", fn, head_dim);
    if (n_heads > 65536) return api_fail(BML_E_UNSUPPORTED, "%s: %u heads", fn, n_heads);
    if (bml_status st = check_pages(page_size, max_pages, fn)) return st;
    if ((uint64_t)n_pages * page_size >= (1ull << 31)) return api_fail(BML_E_INVALID, "%s: %u pages of %u positions", fn, n_pages, page_size);
    if (mask && (n_words < 1 || n_words > bml::kTreeMaxNodes / 64)) return api_fail(BML_E_INVALID, "%s: %u mask words (1 to 4)", fn, n_words);
    if (isnan(scale) || isinf(scale * 1.4426950f)) return api_fail(BML_E_INVALID, "%s: scale is not finite", fn);
    if (bml_status st = ints(fn, {block_table, kv_lens, node_start})) return st;
    if (n_tokens == 0) return bml::api_ok();
    if (n_tokens > 0x7fffffffu) return api_fail(BML_E_INVALID, "%s: %u tokens", fn, n_tokens);
    if (!q_dev || !k_pool || !v_pool || !out_dev || !workspace) return api_fail(BML_E_INVALID, "%s: null pointer", fn);
    if (!aligned(q_dev, 16) || !aligned(out_dev, 16) || !aligned(k_pool, 16) || !aligned(v_pool, 16) || !aligned(workspace, 16) ||
        !aligned(mask, 8))
        return api_fail(BML_E_INVALID, "%s: pointers must be 16-byte aligned (mask 8)", fn);
    const int sms = sm_count(this_device());
    const size_t parts = bml::tree_workspace_bytes(head_dim, sms) * (chunk ? bml::chunk_phases(n_tokens) : 1);
    const size_t need = parts + (chunk ? bml::chunk_work_bytes(n_tokens, n_seqs, sms) : 0);
    if (workspace_bytes < need) return api_fail(BML_E_INVALID, "%s: workspace of %zu bytes, need %zu", fn, workspace_bytes, need);
    const size_t es = bml::dtype_size(q_dtype);
    const uintptr_t qa = reinterpret_cast<uintptr_t>(q_dev), oa = reinterpret_cast<uintptr_t>(out_dev);
    if ((qa < oa ? oa - qa : qa - oa) < (uint64_t)n_tokens * n_heads * head_dim * es)
        return api_fail(BML_E_INVALID, "%s: out overlaps q", fn);
    const uint64_t qb = (uint64_t)n_tokens * n_heads * head_dim * es, n4 = 4ull * n_seqs;
    const uint64_t pool = (uint64_t)n_pages * page_size * n_kv_heads * head_dim * bml::dtype_size(kv_dtype);
    const std::initializer_list<Span> written = {{out_dev, qb}, {workspace, need}};
    if (overlap(written, {{q_dev, qb}, {k_pool, pool}, {v_pool, pool}, {block_table, n4 * max_pages}, {kv_lens, n4}, {node_start, n4 + 4},
                          {mask, 8ull * n_tokens * n_words}}) ||
        overlap(written))
        return api_fail(BML_E_INVALID, "%s: out and workspace must not overlap one another or what is read", fn);
    bml::TreeArgs a = {};
    a.D = head_dim;
    a.kv_type = kv_dtype;
    a.num_sms = sms;
    bml::TreeParams &p = a.p;
    p.q_type = q_dtype;
    bml::tree_rows(a, n_tokens, n_heads / n_kv_heads, n_seqs, n_live, max_nodes);
    a.max_new = max_nodes;
    p.q = q_dev;
    p.out = out_dev;
    p.k = k_pool;
    p.v = v_pool;
    p.node_start = node_start;
    p.node_end = node_start + 1;
    p.mask = mask;
    p.n_tokens = n_tokens;
    p.n_heads = n_heads;
    p.n_kv = n_kv_heads;
    p.group = n_heads / n_kv_heads;
    p.max_pages = max_pages;
    p.n_pages = n_pages;
    p.page_shift = (uint32_t)page_shift(page_size);
    p.n_words = n_words;
    const double sc = scale < 0.f ? 1.0 / sqrt((double)head_dim) : (double)scale;
    p.scale_log2 = (float)(sc * 1.4426950408889634);
    p.part = static_cast<float *>(workspace);
    p.wait_ns = wait_ns;
    p.diag = diag;
    if (chunk) {
        p.n_seqs = n_seqs;
        p.table = block_table;
        p.kv_lens = kv_lens;
        const cudaError_t e = bml::launch_chunk(a, reinterpret_cast<int32_t *>(static_cast<char *>(workspace) + parts), static_cast<cudaStream_t>(stream));
        return e == cudaSuccess ? bml::api_ok() : bml::api_cuda_fail(e, fn);
    }
    for (uint32_t base = 0; base < n_seqs; base += bml::kTreeMaxSeqs) {
        p.n_seqs = n_seqs - base < bml::kTreeMaxSeqs ? n_seqs - base : bml::kTreeMaxSeqs;
        p.table = block_table + (size_t)base * max_pages;
        p.kv_lens = kv_lens + base;
        p.node_start = node_start + base;
        p.node_end = p.node_start + 1;
        const cudaError_t e = bml::launch_tree(a, static_cast<cudaStream_t>(stream));
        if (e != cudaSuccess) return bml::api_cuda_fail(e, fn);
    }
    return bml::api_ok();
}

}  // namespace

BML_API bml_status bml_attn_tree(const void *q_dev, bml_dtype q_dtype, uint32_t n_tokens, uint32_t n_heads,
                                 uint32_t n_kv_heads, uint32_t head_dim, const void *k_pool, const void *v_pool,
                                 bml_dtype kv_dtype, uint32_t n_pages, uint32_t page_size, const int32_t *block_table,
                                 uint32_t max_pages, const int32_t *kv_lens, const int32_t *node_start, uint32_t n_seqs,
                                 const uint64_t *mask, uint32_t n_words, float scale, void *out_dev, void *workspace,
                                 size_t workspace_bytes, void *stream) {
    return attn_tree("bml_attn_tree", false, q_dev, q_dtype, n_tokens, n_heads, n_kv_heads, head_dim, k_pool, v_pool, kv_dtype, n_pages,
                     page_size, block_table, max_pages, kv_lens, node_start, n_seqs, mask, n_words, scale, out_dev, workspace,
                     workspace_bytes, 0u, 0u, bml::kWaitNs, 0u, stream);
}

BML_API bml_status bml_attn_tree_sized(const void *q_dev, bml_dtype q_dtype, uint32_t n_tokens, uint32_t n_heads,
                                       uint32_t n_kv_heads, uint32_t head_dim, const void *k_pool, const void *v_pool,
                                       bml_dtype kv_dtype, uint32_t n_pages, uint32_t page_size, const int32_t *block_table,
                                       uint32_t max_pages, const int32_t *kv_lens, const int32_t *node_start, uint32_t n_seqs,
                                       const uint64_t *mask, uint32_t n_words, float scale, void *out_dev, void *workspace,
                                       size_t workspace_bytes, uint32_t n_live, uint32_t max_nodes, void *stream) {
    return attn_tree("bml_attn_tree_sized", false, q_dev, q_dtype, n_tokens, n_heads, n_kv_heads, head_dim, k_pool, v_pool, kv_dtype,
                     n_pages, page_size, block_table, max_pages, kv_lens, node_start, n_seqs, mask, n_words, scale, out_dev,
                     workspace, workspace_bytes, n_live, max_nodes, bml::kWaitNs, 0u, stream);
}

BML_API bml_status bml_attn_chunk_workspace_size(uint32_t head_dim, uint32_t n_tokens, uint32_t n_seqs, int32_t device, size_t *bytes) {
    const bml_status st = bml_attn_tree_workspace_size(head_dim, device, bytes);
    if (st == BML_OK) *bytes = *bytes * bml::chunk_phases(n_tokens) + bml::chunk_work_bytes(n_tokens, n_seqs, sm_count(device));
    return st;
}

BML_API bml_status bml_attn_chunk(const void *q_dev, bml_dtype q_dtype, uint32_t n_tokens, uint32_t n_heads,
                                  uint32_t n_kv_heads, uint32_t head_dim, const void *k_pool, const void *v_pool,
                                  bml_dtype kv_dtype, uint32_t n_pages, uint32_t page_size, const int32_t *block_table,
                                  uint32_t max_pages, const int32_t *kv_lens, const int32_t *node_start, uint32_t n_seqs,
                                  float scale, void *out_dev, void *workspace, size_t workspace_bytes, uint32_t n_live,
                                  uint32_t max_new, void *stream) {
    return attn_tree("bml_attn_chunk", true, q_dev, q_dtype, n_tokens, n_heads, n_kv_heads, head_dim, k_pool, v_pool, kv_dtype, n_pages,
                     page_size, block_table, max_pages, kv_lens, node_start, n_seqs, nullptr, 0u, scale, out_dev, workspace,
                     workspace_bytes, n_live, max_new, bml::kWaitNs, 0u, stream);
}

BML_API bml_status bml_diag_attn_chunk(const void *q_dev, bml_dtype q_dtype, uint32_t n_tokens, uint32_t n_heads,
                                       uint32_t n_kv_heads, uint32_t head_dim, const void *k_pool, const void *v_pool,
                                       bml_dtype kv_dtype, uint32_t n_pages, uint32_t page_size, const int32_t *block_table,
                                       uint32_t max_pages, const int32_t *kv_lens, const int32_t *node_start, uint32_t n_seqs,
                                       float scale, void *out_dev, void *workspace, size_t workspace_bytes, uint64_t wait_ns,
                                       uint32_t flags, void *stream) {
    const char *fn = "bml_diag_attn_chunk";
    if (flags & ~BML_DIAG_STALL) return api_fail(BML_E_INVALID, "%s: flags 0x%x", fn, flags);
    return attn_tree(fn, true, q_dev, q_dtype, n_tokens, n_heads, n_kv_heads, head_dim, k_pool, v_pool, kv_dtype, n_pages, page_size,
                     block_table, max_pages, kv_lens, node_start, n_seqs, nullptr, 0u, scale, out_dev, workspace, workspace_bytes,
                     0u, 0u, wait_ns ? wait_ns : bml::kWaitNs, (flags & BML_DIAG_STALL) ? bml::kTreeStall : 0u, stream);
}

BML_API bml_status bml_diag_attn_tree(const void *q_dev, bml_dtype q_dtype, uint32_t n_tokens, uint32_t n_heads,
                                      uint32_t n_kv_heads, uint32_t head_dim, const void *k_pool, const void *v_pool,
                                      bml_dtype kv_dtype, uint32_t n_pages, uint32_t page_size, const int32_t *block_table,
                                      uint32_t max_pages, const int32_t *kv_lens, const int32_t *node_start, uint32_t n_seqs,
                                      const uint64_t *mask, uint32_t n_words, float scale, void *out_dev, void *workspace,
                                      size_t workspace_bytes, uint64_t wait_ns, uint32_t flags, void *stream) {
    const char *fn = "bml_diag_attn_tree";
    if (flags & ~BML_DIAG_STALL) return api_fail(BML_E_INVALID, "%s: flags 0x%x", fn, flags);
    return attn_tree(fn, false, q_dev, q_dtype, n_tokens, n_heads, n_kv_heads, head_dim, k_pool, v_pool, kv_dtype, n_pages, page_size,
                     block_table, max_pages, kv_lens, node_start, n_seqs, mask, n_words, scale, out_dev, workspace, workspace_bytes,
                     0u, 0u, wait_ns ? wait_ns : bml::kWaitNs, (flags & BML_DIAG_STALL) ? bml::kTreeStall : 0u, stream);
}

BML_API bml_status bml_diag_attn_tree_form(bml_dtype q_dtype, bml_dtype kv_dtype, uint32_t n_tokens, uint32_t n_heads,
                                           uint32_t n_kv_heads, uint32_t head_dim, uint32_t page_size, uint32_t max_pages,
                                           uint32_t n_seqs, uint32_t n_live, uint32_t max_nodes, int *form) {
    const char *fn = "bml_diag_attn_tree_form";
    if (!form || page_shift(page_size) < 0 || n_kv_heads == 0 || n_heads % n_kv_heads || n_seqs == 0)
        return api_fail(BML_E_INVALID, "%s: bad argument", fn);
    bml::TreeArgs a = {};
    a.D = head_dim;
    a.kv_type = kv_dtype;
    a.num_sms = sm_count(this_device());
    a.p.q_type = q_dtype;
    a.p.n_kv = n_kv_heads;
    a.p.group = n_heads / n_kv_heads;
    a.p.max_pages = max_pages;
    a.p.page_shift = (uint32_t)page_shift(page_size);
    a.p.scale_log2 = 1.f;
    bml::tree_rows(a, n_tokens, a.p.group, n_seqs, n_live, max_nodes);
    *form = (int)bml::tree_form(a);
    return bml::api_ok();
}

BML_API bml_status bml_paged_commit(void *k_pool, void *v_pool, uint32_t n_layers, uint32_t n_pages, uint32_t page_size,
                                    uint32_t n_kv_heads, uint32_t head_dim, bml_dtype kv_dtype,
                                    const int32_t *block_table, uint32_t max_pages, const int32_t *lens,
                                    const int32_t *kv_lens, const int32_t *node_start, uint32_t n, const int32_t *path,
                                    uint32_t max_path, const int32_t *n_accept, int32_t *lens_out, void *stream) {
    const char *fn = "bml_paged_commit";
    if (!valid_dtype(kv_dtype)) return api_fail(BML_E_INVALID, "%s: unknown dtype", fn);
    if (n_layers == 0 || n_layers > 32767 || n_pages == 0 || n_kv_heads == 0 || head_dim == 0 || n == 0 || max_path == 0)
        return api_fail(BML_E_INVALID, "%s: zero dimension or more than 32767 layers", fn);
    if (max_path > 0x7fffffffu) return api_fail(BML_E_INVALID, "%s: max_path %u", fn, max_path);
    if (bml_status st = check_pages(page_size, max_pages, fn)) return st;
    if ((uint64_t)n_pages * page_size >= (1ull << 31)) return api_fail(BML_E_INVALID, "%s: %u pages of %u positions", fn, n_pages, page_size);
    if (bml_status st = ints(fn, {block_table, lens, kv_lens, node_start, path, n_accept, lens_out})) return st;
    const uint64_t row = (uint64_t)n_kv_heads * head_dim * bml::dtype_size(kv_dtype);
    if (row > 0x7fffffffull) return api_fail(BML_E_INVALID, "%s: a row of %llu bytes", fn, (unsigned long long)row);
    if (!k_pool || !v_pool || !aligned(k_pool, 4) || !aligned(v_pool, 4)) return api_fail(BML_E_INVALID, "%s: null or misaligned pool", fn);
    if (overlap({{lens_out, 4ull * n}}, {{lens, 4ull * n}, {kv_lens, 4ull * n}, {node_start, 4ull * n + 4}, {n_accept, 4ull * n},
                                          {path, 4ull * n * max_path}, {block_table, 4ull * n * max_pages}}))
        return api_fail(BML_E_INVALID, "%s: lens_out needs a buffer of its own", fn);
    const uint64_t pool = (uint64_t)n_layers * n_pages * page_size * row;
    if (overlap({{k_pool, pool}}, {{v_pool, pool}})) return api_fail(BML_E_INVALID, "%s: k_pool and v_pool overlap", fn);
    bml::CommitParams p = {};
    p.k_pool = static_cast<char *>(k_pool);
    p.v_pool = static_cast<char *>(v_pool);
    p.n_layers = n_layers;
    p.n_pages = n_pages;
    p.page_shift = (uint32_t)page_shift(page_size);
    p.max_pages = max_pages;
    p.layer_bytes = (uint64_t)n_pages * page_size * row;
    p.row_bytes = (uint32_t)row;
    p.table = block_table;
    p.lens = lens;
    p.kv_lens = kv_lens;
    p.node_start = node_start;
    p.n = n;
    p.path = path;
    p.max_path = max_path;
    p.n_accept = n_accept;
    p.lens_out = lens_out;
    const cudaError_t e = bml::launch_paged_commit(p, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? bml::api_ok() : bml::api_cuda_fail(e, fn);
}
