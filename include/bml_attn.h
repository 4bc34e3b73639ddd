/*
 * bml_attn.h -- C ABI of the B200 attention / KV-cache library
 * (libbmlattn.so, built from bml_b200/csrc for sm_100a).
 *
 * This is the drop-in boundary for bml's attention hot path.  Each entry
 * point names the reference interface it replaces (paths inside the
 * SugarFreeDoNoSo/bml project).  The reference surface is
 *   crates/compiler/src/kv_cache.rs:25-200  (HashConsedKV, softmax_f32,
 *                                            re-exported at lib.rs:33)
 *   crates/compiler/src/gguf_compiler.rs:1008-1050
 *                                           (attention block of
 *                                            forward_layer_cached, reached
 *                                            from forward_cached :929-962)
 *
 * Conventions
 *  - Every function returns a bml_status and never aborts.  Arguments are
 *    validated on the host before anything is launched; a rejected call
 *    returns BML_E_INVALID (where the Rust code would panic, or where this
 *    library declines a shape the reference silently mis-indexes) and
 *    leaves all outputs untouched.  bml_last_error() gives the reason
 *    (thread-local, valid until the next call on that thread).
 *  - "dev" pointers are CUDA device pointers, "host" pointers are host
 *    memory.  The caller owns every pointer it passes.  The library owns
 *    only the device buffers behind a bml_kv handle.
 *  - `stream` is a cudaStream_t passed as void* (NULL = legacy default
 *    stream).  Device-pointer entry points are asynchronous on that stream;
 *    entry points taking host buffers synchronise before returning.
 *  - Layouts are row-major.  A KV cache or K/V tensor is
 *    [position][kv_head][head_dim] (kv_cache.rs:17); queries and outputs
 *    are [head][head_dim] per token (gguf_compiler.rs:1017-1024).
 *  - Scores are scaled by `scale`; pass a negative scale for the
 *    reference's 1/sqrt(head_dim) (gguf_compiler.rs:1010).
 *  - n_heads must be a multiple of n_kv_heads; q head h reads kv head
 *    h / (n_heads / n_kv_heads) (gguf_compiler.rs:1011,1016).
 */
#ifndef BML_ATTN_H
#define BML_ATTN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef int32_t bml_status;
#define BML_OK            0
#define BML_E_INVALID     1 /* bad argument / shape; nothing launched        */
#define BML_E_CUDA        2 /* a CUDA runtime call failed                    */
#define BML_E_NCCL        3 /* reserved for communicator errors              */
#define BML_E_TIMEOUT     4 /* a bounded device-side wait gave up            */
#define BML_E_OOM         5 /* device allocation failed                      */
#define BML_E_UNSUPPORTED 6 /* valid shape the library has no kernel for    */

typedef enum bml_dtype { BML_F32 = 0, BML_F16 = 1, BML_BF16 = 2 } bml_dtype;

#define BML_WHICH_K 0
#define BML_WHICH_V 1

/* ------------------------------------------------------------------------ */
/* Library                                                                  */
/* ------------------------------------------------------------------------ */

/* Reason for the last non-OK status on this thread ("" if none). */
const char *bml_last_error(void);

/* Library version string. */
const char *bml_version(void);

/* ------------------------------------------------------------------------ */
/* KV cache handle  (HashConsedKV, kv_cache.rs:25-181)                       */
/* ------------------------------------------------------------------------ */

typedef struct bml_kv bml_kv;

typedef struct bml_kv_desc {
    uint32_t n_layers;
    uint32_t n_kv_heads;
    uint32_t head_dim;
    uint32_t max_seq_len;
    bml_dtype dtype; /* storage type of K and V; the reference stores f32 */
    int32_t device;  /* CUDA device ordinal                               */
} bml_kv_desc;

/* HashConsedKV::new (kv_cache.rs:53-72): zero-filled per-layer K and V
 * buffers of max_seq_len * n_kv_heads * head_dim elements each. */
bml_status bml_kv_create(const bml_kv_desc *desc, bml_kv **out);

/* Drop of HashConsedKV: frees the device buffers. NULL is accepted. */
bml_status bml_kv_destroy(bml_kv *kv);

/* store_k / store_v (kv_cache.rs:82-101): writes one head vector from host
 * memory into ring slot pos % max_seq_len and counts the store.  len must
 * be >= head_dim (the reference's copy_from_slice panics otherwise); the
 * first head_dim values are stored, converted to the cache dtype.
 * Synchronous. */
bml_status bml_kv_store(bml_kv *kv, int which, uint32_t layer, uint32_t pos,
                        uint32_t kv_head, const float *host_data, size_t len);

/* load_k / load_v (kv_cache.rs:111-124): copies one head vector (widened
 * to f32) into a caller buffer of head_dim floats.  Synchronous. */
bml_status bml_kv_load(const bml_kv *kv, int which, uint32_t layer,
                       uint32_t pos, uint32_t kv_head, float *host_out);

/* dot_qk (kv_cache.rs:135-141): f32 dot of q (host, q_len floats; the
 * shorter length wins) with K[layer][pos % max][kv_head].  Synchronous. */
bml_status bml_kv_dot_qk(const bml_kv *kv, const float *host_q, size_t q_len,
                         uint32_t layer, uint32_t pos, uint32_t kv_head,
                         float *out);

/* k_stats / v_stats (kv_cache.rs:148-155): (stores, stores, 1.0). */
bml_status bml_kv_stats(const bml_kv *kv, int which, uint64_t *unique,
                        uint64_t *total, double *ratio);

/* byte_size (kv_cache.rs:158-161): bytes of all K and V buffers. */
bml_status bml_kv_byte_size(const bml_kv *kv, uint64_t *out);

/* current_pos / advance / advance_by (kv_cache.rs:168-180). */
bml_status bml_kv_current_pos(const bml_kv *kv, uint32_t *out);
bml_status bml_kv_advance(bml_kv *kv);
bml_status bml_kv_advance_by(bml_kv *kv, uint32_t n);

/* Device address of one layer's K or V buffer
 * ([max_seq_len][n_kv_heads][head_dim] in the cache dtype). */
bml_status bml_kv_layer_ptr(const bml_kv *kv, int which, uint32_t layer,
                            void **dev_out);

/* Device-side store of every kv head of one position (the n_kv_heads
 * store_k/store_v calls of gguf_compiler.rs:994-1006 in one launch).
 * k_dev/v_dev: [n_kv_heads][head_dim] in src_dtype, converted to the cache
 * dtype.  Asynchronous on stream. */
bml_status bml_kv_append(bml_kv *kv, uint32_t layer, uint32_t pos,
                         const void *k_dev, const void *v_dev,
                         bml_dtype src_dtype, void *stream);

/* The projection tail of one token in one launch (gguf_compiler.rs:984-1006
 * with apply_rope_inplace, :1290-1317): RoPE -- interleaved pairs
 * (2i, 2i+1) of each head, angle = pos * 10000^(-2i/head_dim), rotated in
 * f64 -- applied to q in place and to k, then k and v stored into the slot
 * of `pos` like bml_kv_append.  q_dev: [n_heads][head_dim] f32 (n_heads a
 * multiple of n_kv_heads); k_dev (before RoPE), v_dev:
 * [n_kv_heads][head_dim] f32.  Asynchronous on stream. */
bml_status bml_kv_append_rope(bml_kv *kv, uint32_t layer, uint32_t pos,
                              float *q_dev, uint32_t n_heads,
                              const float *k_dev, const float *v_dev,
                              void *stream);

/* ------------------------------------------------------------------------ */
/* Decode attention  (gguf_compiler.rs:1008-1050)                           */
/* ------------------------------------------------------------------------ */

/* The attention block of forward_layer_cached for the token at position
 * pos: every q head attends over K/V positions [0, pos] of `layer`
 * (causal), softmax, P.V.  q_dev: [n_heads][head_dim] f32, out_dev:
 * [n_heads][head_dim] f32.  pos must be < max_seq_len (for the reference's
 * ring wrap past max_seq_len, kv_cache.rs:83, use bml_attn_decode_wrap).
 * Uses the handle's own scratch, so calls on one handle must not overlap in
 * time.  Asynchronous. */
bml_status bml_attn_decode(bml_kv *kv, uint32_t layer, uint32_t pos,
                           uint32_t n_heads, float scale, const float *q_dev,
                           float *out_dev, void *stream);

/* bml_attn_decode for any pos, with the reference's behaviour past the end
 * of the ring: its loop (gguf_compiler.rs:1026-1049) runs over positions
 * 0..pos and reads each through slot p % max_seq_len (kv_cache.rs:83), so
 * once pos >= max_seq_len every slot enters the softmax floor(n / M) or
 * floor(n / M) + 1 times (n = pos + 1, M = max_seq_len; the extra visit for
 * slots below n % M).  Computed as attention over the M slots with each
 * slot's weight scaled by its visit count: two KV-split partials merged
 * with the counts.  pos < max_seq_len is bml_attn_decode itself.  Uses the
 * handle's own scratch (allocated on first use), so calls on one handle
 * must not overlap in time.  Asynchronous. */
bml_status bml_attn_decode_wrap(bml_kv *kv, uint32_t layer, uint32_t pos,
                                uint32_t n_heads, float scale,
                                const float *q_dev, float *out_dev,
                                void *stream);

/* One sequence of a batched decode: a contiguous cache
 * [len][n_kv_heads][head_dim] (K and V), whose query token sits at
 * position len-1 and attends over all len positions. */
typedef struct bml_seq_desc {
    const void *k_dev;
    const void *v_dev;
    uint32_t len;
    uint32_t reserved;
} bml_seq_desc;

/* One decode step's appends for a batch of caller-owned caches (the
 * per-request store_k/store_v of gguf_compiler.rs:994-1006, batched; no
 * reference counterpart -- the reference serves one request at a time):
 * writes row seqs[i].len of sequence i ([capacity][n_kv_heads][head_dim]
 * buffers in kv_dtype, writable, room for that row is the caller's) from
 * k_new_dev / v_new_dev [n_seqs][n_kv_heads][head_dim] in src_dtype.  The
 * caller then advances each len.  Asynchronous on stream. */
bml_status bml_kv_append_batched(const bml_seq_desc *seqs_host, uint32_t n_seqs,
                                 uint32_t n_kv_heads, uint32_t head_dim,
                                 bml_dtype kv_dtype, const void *k_new_dev,
                                 const void *v_new_dev, bml_dtype src_dtype,
                                 void *stream);

/* bml_kv_append_batched with the RoPE of bml_kv_append_rope: sequence i's q
 * rows ([n_seqs][n_heads][head_dim] f32, rotated in place) and its new k row
 * are rotated for position seqs[i].len, then k and v ([n_seqs][n_kv_heads]
 * [head_dim] f32) are stored into row seqs[i].len of its caches.  The
 * per-request RoPE + store of gguf_compiler.rs:984-1006 and :1290-1317 for
 * a whole batch in one launch.  Asynchronous on stream. */
bml_status bml_kv_append_rope_batched(const bml_seq_desc *seqs_host,
                                      uint32_t n_seqs, uint32_t n_heads,
                                      uint32_t n_kv_heads, uint32_t head_dim,
                                      bml_dtype kv_dtype, float *q_dev,
                                      const float *k_new_dev,
                                      const float *v_new_dev, void *stream);

/* Scratch bytes recommended for bml_attn_decode_batched / _partial with
 * n_seqs sequences on `device`: room for the partial results of about 8
 * work chunks per SM.  A smaller workspace down to 2 * n_seqs + (SM count)
 * slots still works (the kernels then cut the work into fewer, larger
 * chunks); below that the call returns BML_E_INVALID. */
bml_status bml_attn_decode_workspace_size(uint32_t n_seqs, uint32_t n_heads,
                                          uint32_t head_dim, int32_t device,
                                          size_t *bytes);

/* Batched split-K flash decoding: for every sequence s, the reference
 * attention block over its whole cache (no reference counterpart as a
 * batch: the reference runs one sequence per forward_cached call).
 *   seqs_host : n_seqs descriptors (host memory)
 *   q_dev     : [n_seqs][n_heads][head_dim] f32
 *   out_dev   : [n_seqs][n_heads][head_dim] f32
 *   workspace : device scratch of bml_attn_decode_workspace_size bytes,
 *               zero-filled before its first use; every call leaves it
 *               ready for the next.  Calls sharing a workspace must not
 *               overlap in time.
 * Asynchronous. */
bml_status bml_attn_decode_batched(const bml_seq_desc *seqs_host,
                                   uint32_t n_seqs, uint32_t n_heads,
                                   uint32_t n_kv_heads, uint32_t head_dim,
                                   bml_dtype kv_dtype, float scale,
                                   const float *q_dev, float *out_dev,
                                   void *workspace, size_t workspace_bytes,
                                   void *stream);

/* Allocation-free variant of bml_attn_decode_batched.  It has no
 * counterpart in the reference.  It is for callers that cannot call
 * cudaMalloc: a host runtime that hands all device memory to its own pool
 * allocator at start-up, or a serving loop in which cudaMalloc's implicit
 * device-wide synchronisation would stall other streams.  It takes no
 * workspace; its scratch is a fixed 4 MiB array in device global memory
 * that every GPU loading this library holds until the process exits, and it
 * allocates nothing itself.  A call whose smallest usable scratch -- partial
 * slots for max(2 * n_seqs + (SM count), (8 / n_kv_heads) * n_seqs) results of n_heads rows
 * of head_dim + 2 floats, plus 72.25 KiB of counters -- is above 4 MiB (e.g.
 * 256 sequences of 64 heads at head_dim 128) returns BML_E_INVALID; below
 * that the kernels size their work to the slots the array holds.  The
 * first call on a device looks up the array's device address
 * (cudaGetSymbolAddress); make that first call before any stream capture.
 * All calls share the one array, which keeps the last call's contents: each
 * call first clears the schedule counters on `stream`, so calls that
 * overlap in time on the GPU race with each other and must be serialised
 * (one stream, or events between streams).  The array's error word is not
 * cleared by a call: a bounded device wait that gave up stays recorded
 * until bml_attn_noalloc_check reads it.  Results agree with
 * bml_attn_decode_batched's within the decode tolerance.  Asynchronous. */
bml_status bml_attn_decode_batched_noalloc(const bml_seq_desc *seqs_host,
                                           uint32_t n_seqs, uint32_t n_heads,
                                           uint32_t n_kv_heads, uint32_t head_dim,
                                           bml_dtype kv_dtype, float scale,
                                           const float *q_dev, float *out_dev,
                                           void *stream);

/* Reads and clears the error word of the fixed scratch array of
 * bml_attn_decode_batched_noalloc on the current device: BML_E_TIMEOUT if a
 * bounded device wait of an earlier call gave up (that call's output is not
 * valid), else BML_OK.  Like the entry point it serves, it has no
 * counterpart in the reference and allocates nothing.  Synchronises
 * `stream`. */
bml_status bml_attn_noalloc_check(void *stream);

/* KV-split partial: the same computation over each sequence's slice of the
 * cache, returning per (sequence, q head) the running max m (in log2
 * units: max over positions of scale*log2(e)*q.k), the softmax
 * denominator l relative to m, and the normalised partial output
 * o = sum_p 2^(s_p - m) v_p / l.  Partials from disjoint slices of one
 * cache merge exactly with bml_attn_merge_lse.
 *   m_dev, l_dev : [n_seqs][n_heads] f32;  o_dev : [n_seqs][n_heads][head_dim]
 * Asynchronous. */
bml_status bml_attn_decode_partial(const bml_seq_desc *seqs_host,
                                   uint32_t n_seqs, uint32_t n_heads,
                                   uint32_t n_kv_heads, uint32_t head_dim,
                                   bml_dtype kv_dtype, float scale,
                                   const float *q_dev, float *m_dev,
                                   float *l_dev, float *o_dev,
                                   void *workspace, size_t workspace_bytes,
                                   void *stream);

/* Log-sum-exp merge of n_parts partial triples (as written by
 * bml_attn_decode_partial, stacked along a leading part axis):
 *   m_dev, l_dev : [n_parts][n_rows];  o_dev : [n_parts][n_rows][head_dim]
 *   out_dev      : [n_rows][head_dim] f32
 * out = sum_i 2^(m_i-M) l_i o_i / sum_i 2^(m_i-M) l_i with M = max_i m_i,
 * summed in part order.  Asynchronous. */
bml_status bml_attn_merge_lse(const float *m_dev, const float *l_dev,
                              const float *o_dev, uint32_t n_parts,
                              uint32_t n_rows, uint32_t head_dim,
                              float *out_dev, void *stream);

/* The same merge over partials packed one part after another as
 * [m (n_rows) | l (n_rows) | o (n_rows*head_dim)] -- the layout an
 * all-gather of one packed buffer per GPU produces (KV split across GPUs).
 * Asynchronous. */
bml_status bml_attn_merge_lse_packed(const float *parts_dev, uint32_t n_parts,
                                     uint32_t n_rows, uint32_t head_dim,
                                     float *out_dev, void *stream);

/* ------------------------------------------------------------------------ */
/* Causal prefill  (gguf_compiler.rs:946-958 token loop over :1008-1050)     */
/* ------------------------------------------------------------------------ */

/* Attention for every token of n_seqs prompts of seq_len tokens at once:
 * token t of a sequence attends over positions [0, t] of that sequence
 * (causal != 0) or over all positions (causal == 0).  Tensor-core
 * (tcgen05) kernel: q/k/v are 16-bit (in_dtype BML_BF16 or BML_F16),
 * accumulation is f32.
 *   q_dev   : [n_seqs][seq_len][n_heads][head_dim]
 *   k_dev, v_dev : [n_seqs][seq_len][n_kv_heads][head_dim]
 *   out_dev : [n_seqs][seq_len][n_heads][head_dim] in out_dtype
 *             (BML_F32 or in_dtype)
 * head_dim 64 or 128.  Asynchronous. */
bml_status bml_attn_prefill(const void *q_dev, const void *k_dev,
                            const void *v_dev, uint32_t n_seqs,
                            uint32_t seq_len, uint32_t n_heads,
                            uint32_t n_kv_heads, uint32_t head_dim,
                            bml_dtype in_dtype, float scale, int causal,
                            void *out_dev, bml_dtype out_dtype, void *stream);

/* ------------------------------------------------------------------------ */
/* softmax_f32 (kv_cache.rs:188-200)                                        */
/* ------------------------------------------------------------------------ */

/* Row-wise softmax_f32 of n_rows rows of n floats: max-subtracted exp,
 * divided by the row sum, and uniform 1/n where the sum is not positive.
 * n == 0 is valid and does nothing (the reference returns an empty Vec).
 * Asynchronous. */
bml_status bml_softmax_f32(const float *x_dev, uint32_t n_rows, uint32_t n,
                           float *out_dev, void *stream);

/* ------------------------------------------------------------------------ */
/* KV split of one sequence over GPUs                                       */
/* ------------------------------------------------------------------------ */

/* One long sequence whose KV cache is cut into contiguous slices, one per
 * GPU (one process per GPU).  No reference counterpart: the reference runs
 * the whole loop of gguf_compiler.rs:1026-1049 in one thread.  Every rank
 * decodes its slice and, inside the same kernel, exchanges per-(q head, 32
 * dims) partials (max, sum, normalised output) with every other rank over
 * peer memory (CUDA IPC mappings, plain loads and stores) and merges them
 * in rank order with the log-sum-exp rule; every rank ends with the same
 * output.  Set-up: bml_kvsplit_create on each rank, bml_kvsplit_handle ->
 * BML_KVSPLIT_HANDLE_BYTES bytes, gathered from all ranks in rank order
 * (any host channel), bml_kvsplit_open.  All ranks must then call
 * bml_attn_decode_kvsplit the same number of times with the same shape;
 * a rank whose peers do not arrive within 2 s stops waiting and records
 * BML_E_TIMEOUT in the workspace's error word (bml_attn_workspace_check).
 * The calls' exchange epochs are counted on the device (in the exchange
 * buffer, advanced by each launch), so the calls may be captured in a CUDA
 * graph and replayed, on every rank alike. */
typedef struct bml_kvsplit bml_kvsplit;
#define BML_KVSPLIT_HANDLE_BYTES 64

bml_status bml_kvsplit_create(int32_t device, uint32_t rank, uint32_t world,
                              uint32_t n_heads, uint32_t head_dim,
                              bml_kvsplit **out);
bml_status bml_kvsplit_handle(const bml_kvsplit *h, void *handle_out,
                              size_t bytes);
bml_status bml_kvsplit_open(bml_kvsplit *h, const void *handles,
                            size_t bytes);
/* slice_host: this rank's slice of the cache (one descriptor, its own
 * positions only); q_dev [n_heads][head_dim] f32, the same on every rank;
 * out_dev [n_heads][head_dim] f32.  16-bit caches with the decode kernel's
 * shapes.  Asynchronous. */
bml_status bml_attn_decode_kvsplit(bml_kvsplit *h, const bml_seq_desc *slice_host,
                                   uint32_t n_heads, uint32_t n_kv_heads,
                                   uint32_t head_dim, bml_dtype kv_dtype,
                                   float scale, const float *q_dev,
                                   float *out_dev, void *workspace,
                                   size_t workspace_bytes, void *stream);
bml_status bml_kvsplit_destroy(bml_kvsplit *h);

/* ------------------------------------------------------------------------ */
/* Paged KV cache and drafted tokens                                        */
/* ------------------------------------------------------------------------ */

/* A paged cache keeps every request's K and V in pages of page_size
 * positions out of one pool per layer, [n_pages][page_size][n_kv_heads]
 * [head_dim] (a row of the pool is one position of all kv heads, the
 * reference's layout, kv_cache.rs:17), and a block table [n][max_pages] of
 * page indices per request.  All sizes of a step -- lengths, new tokens,
 * page counts -- stay on the device, so a step needs no host
 * synchronisation and can be captured in a CUDA graph.  No reference
 * counterpart: the reference keeps one flat buffer per layer and decodes
 * one token at a time.
 *
 * A step of a batch of n requests:
 *   bml_paged_plan      pages for the new tokens, their slots, positions and
 *                       (for drafts) ancestor masks -- once a step
 *   bml_paged_append    RoPE of q and k, K and V rows stored -- every layer
 *   bml_attn_tree       attention of the new tokens -- every layer; or
 *   bml_attn_chunk      the same for any number of them, without drafts
 *   bml_verify_drafts   which drafted tokens the target model keeps
 *   bml_paged_commit    the rows of the accepted path moved to the front,
 *                       all layers, new lengths -- once a step
 * and between steps bml_page_fork (requests that share another's pages),
 * bml_page_free (pages of requests that end or are rolled back) and
 * bml_page_compact (the pool packed to its front).
 * page_size is a power of two from 16 to 1024 and max_pages * page_size
 * below 2^31 in every call. */

/* Plans one step.  Request i has lens[i] committed positions, owned[i] pages
 * in its row of block_table, and n_new[i] new tokens (0 for none); token rows
 * are the requests' new tokens in request order.
 *   free_pages [n_free]: the pool's pages; the first *free_used are taken,
 *       and pages are taken from there on, in request order;
 *   node_start [n+1]: first token row of each request, and the end;
 *   kv_lens [n]: lens + n_new, or 0 for a refused request;
 *   owned_out [n], free_used_out [1]: the counts after this plan;
 *   block_table [n][max_pages]: new entries written, others left;
 *   slots [n_tokens] int64: row of the pool for each token, -1 for a token of
 *       a refused request and for rows behind the last token;
 *   positions [n_tokens]: RoPE position: lens + j for the j-th token, with
 *       parents lens + depth; 0 where the slot is -1;
 *   parents [n_tokens] or NULL: a drafted token's parent among its request's
 *       tokens, -1 (or anything not before the token) for a child of the last
 *       committed token;
 *   mask [n_tokens][n_words] (with parents; n_words 1 to 4): bits of the
 *       token's ancestors and of itself; zero where the slot is -1;
 *   status [n]: 0, or why the request is refused: 1 not enough free pages
 *       (for it and the requests before it), 2 more positions than its table
 *       row holds, more than 64 * n_words drafted tokens, or a negative
 *       count, 4 its tokens lie beyond n_tokens.  A refused request takes no
 *       pages.
 * All arrays are int32 on the device unless noted; results have buffers of
 * their own.  n <= 4096.  Asynchronous. */
bml_status bml_paged_plan(const int32_t *lens, const int32_t *n_new,
                          const int32_t *owned, uint32_t n,
                          const int32_t *free_pages, uint32_t n_free,
                          const int32_t *free_used, uint32_t page_size,
                          uint32_t max_pages, int32_t *block_table,
                          const int32_t *parents, uint32_t n_tokens,
                          uint32_t n_words, int32_t *node_start,
                          int32_t *kv_lens, int32_t *owned_out,
                          int32_t *free_used_out, int64_t *slots,
                          int32_t *positions, uint64_t *mask, int32_t *status,
                          void *stream);

/* RoPE and store of n_tokens tokens of one layer: q [n_tokens][n_heads]
 * [head_dim] turned by positions (interleaved pairs, angle position *
 * theta^(-2i/head_dim), gguf_compiler.rs:1290-1317 with theta 10000) into
 * q_out (q itself, or a buffer that does not overlap it), k turned and v as
 * is ([n_tokens][n_kv_heads][head_dim]) into row slots[t] of the pools.
 * positions NULL: no rotation.  q and q_out NULL: no queries.  A token whose
 * slot is outside [0, n_rows) is skipped: nothing of it is written.  Angles
 * are f64, the rotation f32; results are rounded once to the destination's
 * type.  Slots of one call must differ (of two tokens with the same slot,
 * either's values may be stored), and the two pools, q_out and what is read must
 * not overlap.  head_dim even; pointers aligned to two
 * elements; theta at least 2^-16; negative positions count as 0.
 * Asynchronous. */
bml_status bml_paged_append(const void *q_dev, const void *k_dev,
                            const void *v_dev, bml_dtype src_dtype,
                            const int64_t *slots, const int32_t *positions,
                            uint32_t n_tokens, uint32_t n_heads,
                            uint32_t n_kv_heads, uint32_t head_dim,
                            double theta, void *q_out_dev, void *k_pool,
                            void *v_pool, bml_dtype kv_dtype, uint64_t n_rows,
                            void *stream);

/* Scratch bytes of bml_attn_tree on `device` (whatever the batch). */
bml_status bml_attn_tree_workspace_size(uint32_t head_dim, int32_t device,
                                        size_t *bytes);

/* Attention of every request's new tokens over its pages: token row t of
 * request i (node j = t - node_start[i] of T) attends over the committed
 * positions [0, kv_lens[i] - T) and over those nodes whose bits are set in
 * mask[t]; mask NULL: over nodes 0..j (a chain; T = 1 is plain decode).
 *   node_start: ascending, as bml_paged_plan writes it;
 *   q_dev, out_dev: [n_tokens][n_heads][head_dim] in q_dtype: BML_F32 with
 *       pages of any type, or the pages' own 16-bit type;
 *   workspace: bml_attn_tree_workspace_size bytes, 16-byte aligned, no
 *       contents needed; calls that share one must not overlap in time.  It and
 *       out_dev overlap nothing that the call reads.
 * At most 256 nodes a request (64 * n_words with a mask).  Rows that see
 * nothing are zero; so are all rows of a request with kv_lens[i] < T (one
 * that bml_paged_plan refused), with more nodes than that, or with more
 * positions than its table holds.  Positions on a page outside [0, n_pages)
 * count as masked.  What lies in masked places -- cache rows past kv_lens,
 * nodes that a row does not see, infinities and NaN among them -- does not
 * reach the row.  An infinity in V that a row does see makes that column of the
 * row infinite (NaN beside one of the other sign), whatever its weight.
 * Token rows outside the requests' are left as they were.
 * Sums are divided by the weights' sum at the end: where 2^8 times the sum of |v|
 * that a row sees leaves f32's range, that column is infinite or NaN.
 * 16-bit queries: scores and sums in f32, the softmax weights rounded to the
 * 16-bit type before P.V, one rounding of the output; 32-bit queries: about
 * f32 precision throughout (over f16 pages a weight has steps of 2^-44 of the
 * row's largest).  Results are the same from run to run on one
 * device.  Should a wait inside a kernel run into its limit (2 s), the rows that
 * its CTA had not written yet become NaN.  head_dim 64 or 128.  Asynchronous. */
bml_status bml_attn_tree(const void *q_dev, bml_dtype q_dtype,
                         uint32_t n_tokens, uint32_t n_heads,
                         uint32_t n_kv_heads, uint32_t head_dim,
                         const void *k_pool, const void *v_pool,
                         bml_dtype kv_dtype, uint32_t n_pages,
                         uint32_t page_size, const int32_t *block_table,
                         uint32_t max_pages, const int32_t *kv_lens,
                         const int32_t *node_start, uint32_t n_seqs,
                         const uint64_t *mask, uint32_t n_words, float scale,
                         void *out_dev, void *workspace,
                         size_t workspace_bytes, void *stream);

/* bml_attn_tree for a caller that knows more of its batch: n_live requests have
 * new tokens (0: not known, all n_seqs), the most of one are max_nodes (0: not
 * known, the average).  The kernel is chosen by them, where bml_attn_tree has
 * only the average over all n_seqs; results are right whatever they say. */
bml_status bml_attn_tree_sized(const void *q_dev, bml_dtype q_dtype,
                               uint32_t n_tokens, uint32_t n_heads,
                               uint32_t n_kv_heads, uint32_t head_dim,
                               const void *k_pool, const void *v_pool,
                               bml_dtype kv_dtype, uint32_t n_pages,
                               uint32_t page_size, const int32_t *block_table,
                               uint32_t max_pages, const int32_t *kv_lens,
                               const int32_t *node_start, uint32_t n_seqs,
                               const uint64_t *mask, uint32_t n_words,
                               float scale, void *out_dev, void *workspace,
                               size_t workspace_bytes, uint32_t n_live,
                               uint32_t max_nodes, void *stream);

/* Scratch bytes of bml_attn_chunk on `device` for a batch of that size. */
bml_status bml_attn_chunk_workspace_size(uint32_t head_dim, uint32_t n_tokens,
                                         uint32_t n_seqs, int32_t device,
                                         size_t *bytes);

/* Attention of chunks of new tokens over pages: bml_attn_tree without a mask,
 * for any number of new tokens a request -- a prompt or a part of one, beside
 * requests that decode one token.  Token row t of request i (the j-th of its T,
 * j = t - node_start[i]) attends over the positions [0, kv_lens[i] - T + j].
 * Types, layouts, refused requests, masked places, infinities, precision and the
 * limit of waits are bml_attn_tree's (for values of normal distribution, results of
 * 16-bit queries are off by 2.3e-3 of their norm with bf16 and 2.8e-4 with f16, where
 * the rounding of the result alone makes 1.7e-3 and 2.1e-4: the weights' rounding
 * makes the rest; of 32-bit queries by 6e-7).  workspace:
 * bml_attn_chunk_workspace_size bytes, 16-byte aligned, no contents needed, not
 * shared by calls that overlap in time; for batches of 1024 tokens and more four times
 * bml_attn_tree's and a little (on a B200 158 MB with head_dim 128, 80 MB with 64),
 * whatever the types, else once.  n_live, max_new: as bml_attn_tree_sized's n_live and
 * max_nodes, 0 where not known; the choice of a kernel goes by them.
 * bml_attn_tree_sized is the faster call for more than 8 requests of a token each
 * (bf16, head_dim 128, 32 of them behind 1000 positions: 28 us and 38; behind 30,000:
 * 582 and 612); from about 64 tokens a request on this one mostly is (8 of 64 behind
 * 1000: 48 us and 35; 16 of 256: 176 and 126, but behind 8000 581 and 603; f32 queries
 * over bf16 pages, 8 of 64 behind 8000: 758 and 417).  head_dim 64 or 128.
 * Asynchronous. */
bml_status bml_attn_chunk(const void *q_dev, bml_dtype q_dtype,
                          uint32_t n_tokens, uint32_t n_heads,
                          uint32_t n_kv_heads, uint32_t head_dim,
                          const void *k_pool, const void *v_pool,
                          bml_dtype kv_dtype, uint32_t n_pages,
                          uint32_t page_size, const int32_t *block_table,
                          uint32_t max_pages, const int32_t *kv_lens,
                          const int32_t *node_start, uint32_t n_seqs,
                          float scale, void *out_dev, void *workspace,
                          size_t workspace_bytes, uint32_t n_live,
                          uint32_t max_new, void *stream);

/* Verification of drafted tokens: which path of each request's draft is kept,
 * and the token that follows it, so that tokens are distributed as the target
 * model's.  Nodes are those of bml_paged_plan: token row t of request i is node
 * j = t - node_start[i]; node 0 is the pending token (chosen before, not in the
 * cache yet) and is always kept; a node whose parent is an earlier node of its
 * request is a drafted child of that node, any other never kept.
 *   target [n_tokens][vocab]: the target model's probabilities behind each node;
 *   draft [n_tokens][vocab]: those that each node's children were drawn from,
 *       independently of one another (rows of nodes without children are not
 *       read); NULL: the tokens were picked, not drawn (the likeliest ones);
 *   u [n_tokens], u_next [n]: random numbers, uniform in [0, 1);
 *   path [n][max_path], n_accept [n]: the kept nodes in order, as
 *       bml_paged_commit takes them; -1 behind them;
 *   next [n]: the token behind the path, the next step's pending token.
 * At a kept node with rows p and q its children are tried in node order: the
 * k-th, of token x, is kept if u q(x) S_k < max(p(x) - c_k q(x), 0), where
 * c_0 = 0, S_0 = 1, and after a rejection c_(k+1) = c_k + S_k, S_(k+1) =
 * sum_v max(p(v) - c_(k+1) q(v), 0).  If none is, the path ends there and next
 * is the smallest v with C(v) > u_next * C(vocab - 1), C the prefix sums of
 * max(p - c q, 0) with the last c.  Without draft: kept if u S < p(x), and a
 * rejected x leaves p (S loses p(x), and it is neither kept nor drawn).  Where
 * nothing of positive weight is left, which rounding can do to 16-bit rows, next
 * is drawn from p itself; if p has nothing either, or q sums to more than twice p
 * (no distribution: nothing can be said of the token then), it is vocab - 1.  Sums are
 * f64.  A path of max_path nodes ends there, its last node's children untried.  Probabilities that are not positive finite numbers
 * count as 0; a child whose token is outside [0, vocab) is never tried.  A request
 * without nodes, or with more than 256, has n_accept 0 and next -1.  A request
 * that bml_paged_plan refused is walked like any other, though its attention was
 * zero: bml_paged_commit keeps nothing of it, and its results here mean nothing.
 * target and draft are of one type, rows need no alignment beyond it.
 * Asynchronous. */
bml_status bml_verify_drafts(const void *target, const void *draft,
                             bml_dtype dtype, uint32_t vocab,
                             const int32_t *tokens, const int32_t *parents,
                             uint32_t n_tokens, const int32_t *node_start,
                             uint32_t n, const float *u, const float *u_next,
                             uint32_t max_path, int32_t *path,
                             int32_t *n_accept, int32_t *next, void *stream);

/* Commits the accepted path of every request's draft: in the K and V pools of
 * all n_layers layers (layer l at pool + l * n_pages * page_size * row), row
 * lens[i] + path[i][k] moves to row lens[i] + k for k < n_accept[i], and
 * lens_out[i] = lens[i] + the accepted count.  path [n][max_path] int32 holds
 * strictly increasing node indices; an entry that is not larger than the one
 * before, or not below the request's node count, ends the path there, and the
 * count with it.  A request with kv_lens[i] != lens[i] + its node count (one
 * that the plan refused) commits nothing.  lens_out is its own buffer, and the
 * two pools must not overlap.
 * Asynchronous. */
bml_status bml_paged_commit(void *k_pool, void *v_pool, uint32_t n_layers,
                            uint32_t n_pages, uint32_t page_size,
                            uint32_t n_kv_heads, uint32_t head_dim,
                            bml_dtype kv_dtype, const int32_t *block_table,
                            uint32_t max_pages, const int32_t *lens,
                            const int32_t *kv_lens, const int32_t *node_start,
                            uint32_t n, const int32_t *path, uint32_t max_path,
                            const int32_t *n_accept, int32_t *lens_out,
                            void *stream);

/* Pages held by several requests.  shared [n_pages] int32 counts a page's
 * holders beyond the first (0: one holder, or none), so bml_paged_plan's new
 * pages need no entry: an array of zeros at the start.  Shared pages are full
 * ones, behind which nobody writes: a request's part-filled page is always its
 * own.  The calls below, like the plan, leave lens, owned, shared and the free
 * list's count as they are and write their next values into buffers of their
 * own, which must not overlap one another or what is read.  n, m <= 4096.
 *
 * Forks: row dst[j] of the tables continues the lens[src[j]] positions of row
 * src[j] (several samples of one prompt, beams).  Full pages are shared; the rows
 * of a part-filled one are copied in all layers to a page of the free list, taken
 * in the order of j.  dst must be an idle row (lens and owned 0).
 *   block_table: row dst[j] written, nothing else;
 *   lens_out, owned_out [n], shared_out [n_pages], free_used_out [1];
 *   status [m]: 0, or why fork j is refused: 1 not enough free pages (for it and
 *       the forks before it), 2 a row outside [0, n), a dst that is not idle or
 *       that an earlier fork names, or a src whose pages do not hold its positions.
 *       A refused fork changes nothing.
 * Layers lie as in bml_paged_commit.  Asynchronous. */
bml_status bml_page_fork(void *k_pool, void *v_pool, uint32_t n_layers,
                         uint32_t n_pages, uint32_t page_size,
                         uint32_t n_kv_heads, uint32_t head_dim,
                         bml_dtype kv_dtype, const int32_t *src,
                         const int32_t *dst, uint32_t m, const int32_t *lens,
                         const int32_t *owned, uint32_t n,
                         int32_t *block_table, uint32_t max_pages,
                         const int32_t *shared, const int32_t *free_pages,
                         uint32_t n_free, const int32_t *free_used,
                         int32_t *lens_out, int32_t *owned_out,
                         int32_t *shared_out, int32_t *free_used_out,
                         int32_t *status, void *stream);

/* Ends or rolls back requests: request i keeps min(lens[i], keep[i]) positions
 * and the pages that hold them, and releases the pages behind (0: all of them;
 * its length or more: spare pages only; negative: it is left as it is).  A page
 * that all its holders have released is free again.
 *   free_out [n_free]: free_pages with the taken part [0, *free_used) parted into
 *       the pages that are still held and, behind *free_used_out, the freed ones,
 *       each in the order they had;
 *   lens_out, owned_out [n], shared_out [n_pages], free_used_out [1];
 *   status [n]: 8 where keep ends inside a page that others hold: the request is
 *       left as it is (its next token would be written there); else 0.
 * block_table is not written: entries from owned_out on mean nothing.
 * workspace: 4096 + 4 * ceil(n_free / 32) bytes, no contents needed, not shared by
 * calls that overlap in time.  Asynchronous. */
bml_status bml_page_free(const int32_t *keep, const int32_t *lens,
                         const int32_t *owned, uint32_t n,
                         const int32_t *block_table, uint32_t max_pages,
                         uint32_t page_size, const int32_t *shared,
                         uint32_t n_pages, const int32_t *free_pages,
                         uint32_t n_free, const int32_t *free_used,
                         int32_t *lens_out, int32_t *owned_out,
                         int32_t *shared_out, int32_t *free_out,
                         int32_t *free_used_out, int32_t *status,
                         void *workspace, size_t workspace_bytes, void *stream);

/* Packs a pool: the H held pages (the first owned[i] entries of each table row)
 * come to lie at [0, H), in all layers.  Held pages from H on move, in ascending
 * order, into the pages below H that nobody holds, in ascending order; the
 * others stay.  The tables (table_out [n][max_pages], other entries copied) and
 * shared counts (shared_out [n_pages], 0 for free pages) follow, free_out
 * [n_pages] becomes 0, 1, 2, ... and free_used_out H: the free list is that of
 * the whole pool.  Pages from H on keep what they held.  workspace: 12 * n_pages
 * + 4 bytes, no contents needed, not shared by calls that overlap in time.
 * Asynchronous. */
bml_status bml_page_compact(void *k_pool, void *v_pool, uint32_t n_layers,
                            uint32_t n_pages, uint32_t page_size,
                            uint32_t n_kv_heads, uint32_t head_dim,
                            bml_dtype kv_dtype, const int32_t *owned,
                            uint32_t n, const int32_t *block_table,
                            uint32_t max_pages, const int32_t *shared,
                            int32_t *table_out, int32_t *shared_out,
                            int32_t *free_out, int32_t *free_used_out,
                            void *workspace, size_t workspace_bytes,
                            void *stream);

/* ------------------------------------------------------------------------ */
/* Device-side error word                                                   */
/* ------------------------------------------------------------------------ */

/* Reads and clears the error word kernels set in a decode workspace when a
 * bounded wait gives up.  Returns BML_OK or BML_E_TIMEOUT.  Synchronises
 * the stream. */
bml_status bml_attn_workspace_check(void *workspace, size_t workspace_bytes,
                                    void *stream);

#ifdef __cplusplus
}
#endif

#endif /* BML_ATTN_H */
