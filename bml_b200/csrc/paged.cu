// paged.cu -- the paged KV cache's bookkeeping and row kernels: page
// planning (block tables, slots, ancestor masks), RoPE append through slots,
// and the commit of an accepted path.
//
// The reference keeps one flat buffer per layer (crates/compiler/src/
// kv_cache.rs:25-181 in SugarFreeDoNoSo/bml) and stores one token at a time
// (gguf_compiler.rs:984-1006); pages, drafted tokens and their commit have no
// counterpart there.
#include <math.h>

#include "paged.cuh"

namespace bml {

namespace {

// ---------------------------------------------------------------------------
// Block-wide exclusive scan of one 64-bit value per thread
// ---------------------------------------------------------------------------
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t *warp_sums, int64_t *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    int64_t inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
    }
    if (lane == 31) warp_sums[warp] = inc;
    __syncthreads();
    int64_t before = 0, all = 0;
    for (int w = 0; w < nw; ++w) {
        const int64_t s = warp_sums[w];
        before += w < warp ? s : 0;
        all += s;
    }
    __syncthreads();
    *total = all;
    return before + inc - v;
}

// ---------------------------------------------------------------------------
// page_plan
//
//   need_i = ceil((len_i + new_i) / page), add_i = max(0, need_i - owned_i),
//   base_i = used + sum of add over the requests before i,
//   table[i][owned_i + j] = free[base_i + j],
//   token j of request i: position len_i + j, slot = its row in the pool.
//
// Every CTA redoes the two prefix sums over the requests (a few loads a
// thread; cheaper than a second launch) and then takes its share of table
// entries and tokens; entries that this plan adds are computed from the free
// list, never read back, so the CTAs need not wait for one another.
// ---------------------------------------------------------------------------
constexpr int kPlanThreads = 256;

__global__ void __launch_bounds__(kPlanThreads) page_plan_kernel(const PlanParams p) {
    extern __shared__ int32_t sh[];
    int32_t *s_start = sh;                 // [n + 1] first token
    int32_t *s_base = sh + p.n + 1;        // [n] first new page's place in the free list
    int32_t *s_own = s_base + p.n;         // [n] pages held before, or -1: refused
    __shared__ int64_t warp_sums[kPlanThreads / 32];
    const uint32_t per = (p.n + kPlanThreads - 1) / kPlanThreads;
    const uint32_t i0 = min(threadIdx.x * per, p.n), i1 = min(i0 + per, p.n);
    const int64_t ps = 1ll << p.page_shift;

    int64_t tok = 0;
    for (uint32_t i = i0; i < i1; ++i) tok += max(p.n_new[i], 0);
    int64_t all_tok;
    int64_t at = block_scan(tok, warp_sums, &all_tok);
    const int64_t first_tok = at;
    // pages: requests that are bad or whose tokens do not fit take none
    auto judge = [&](uint32_t i, int64_t end, int64_t &add) {
        const int64_t len = p.lens[i], nw = p.n_new[i], own = p.owned[i];
        const int64_t need = (len + nw + ps - 1) >> p.page_shift;
        add = 0;
        if (len < 0 || nw < 0 || own < 0 || own > p.max_pages || need > p.max_pages ||
            (p.parents && nw > 64ll * p.n_words))
            return kPlanBad;
        if (end > p.n_tokens) return kPlanNoRoom;
        add = need > own ? need - own : 0;
        return 0;
    };
    int64_t pages = 0;
    for (uint32_t i = i0; i < i1; ++i) {
        int64_t add;
        at += max(p.n_new[i], 0);
        judge(i, at, add);
        pages += add;
    }
    int64_t all_pages;
    int64_t cum = block_scan(pages, warp_sums, &all_pages);
    const int64_t used = min(max(*p.free_used, 0), (int32_t)p.n_free);
    const int64_t avail = (int64_t)p.n_free - used;
    int64_t granted = 0;  // largest running sum that still fits
    at = first_tok;
    for (uint32_t i = i0; i < i1; ++i) {
        int64_t add;
        const int64_t begin = at;
        at += max(p.n_new[i], 0);
        int32_t st = judge(i, at, add);
        const int64_t base = cum;
        cum += add;
        if (st == 0 && add > 0) {
            if (cum > avail) st = kPlanNoPages;
            else granted = cum;
        }
        s_start[i] = (int32_t)min(begin, (int64_t)p.n_tokens);
        s_base[i] = (int32_t)min(used + base, (int64_t)p.n_free);
        s_own[i] = st ? -1 : p.owned[i];
        if (blockIdx.x == 0) {
            p.node_start[i] = s_start[i];
            p.kv_lens[i] = st ? 0 : p.lens[i] + p.n_new[i];
            p.owned_out[i] = p.owned[i] + (st ? 0 : (int32_t)add);
            p.status[i] = st;
        }
    }
    if (threadIdx.x == 0) s_start[p.n] = (int32_t)min(all_tok, (int64_t)p.n_tokens);
    if (blockIdx.x == 0) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const int64_t u = __shfl_xor_sync(0xffffffffu, granted, o);
            granted = granted > u ? granted : u;
        }
        if ((threadIdx.x & 31) == 0) warp_sums[threadIdx.x >> 5] = granted;
    }
    __syncthreads();
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        p.node_start[p.n] = s_start[p.n];
        int64_t g = 0;
        for (int w = 0; w < kPlanThreads / 32; ++w) g = g > warp_sums[w] ? g : warp_sums[w];
        *p.free_used_out = (int32_t)(used + g);
    }

    // new table entries: a warp per request
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t gw = blockIdx.x * (kPlanThreads / 32) + (threadIdx.x >> 5), n_warps = gridDim.x * (kPlanThreads / 32);
    for (uint32_t i = gw; i < p.n; i += n_warps) {
        const int32_t own = s_own[i];
        if (own < 0) continue;
        const int64_t need = ((int64_t)p.lens[i] + p.n_new[i] + ps - 1) >> p.page_shift;
        for (int64_t j = own + (int64_t)lane; j < need; j += 32)
            p.table[(size_t)i * p.max_pages + j] = p.free_pages[s_base[i] + (j - own)];
    }

    // tokens
    const int32_t total = s_start[p.n];
    for (uint32_t t = blockIdx.x * kPlanThreads + threadIdx.x; t < p.n_tokens; t += gridDim.x * kPlanThreads) {
        int64_t slot = -1;
        int32_t rope = 0;
        uint64_t m[kTreeMaxNodes / 64] = {0, 0, 0, 0};
        if ((int32_t)t < total) {
            // the last request that starts at or before t (empty ones in between have the same start)
            uint32_t lo = 0, hi = p.n;
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) >> 1;
                if (s_start[mid] <= (int32_t)t) lo = mid;
                else hi = mid;
            }
            const int32_t own = s_own[lo], j = (int32_t)t - s_start[lo];
            if (own >= 0) {
                const int64_t pos = (int64_t)p.lens[lo] + j;
                const int64_t pg = pos >> p.page_shift;
                const int64_t page = pg < own ? p.table[(size_t)lo * p.max_pages + pg] : p.free_pages[s_base[lo] + (pg - own)];
                slot = (page << p.page_shift) + (pos & (ps - 1));
                rope = (int32_t)pos;
                if (p.parents) {
                    // up the tree; a parent that is not an earlier node ends the walk (a root)
                    int32_t a = j, depth = 0;
                    while (true) {
                        m[a >> 6] |= 1ull << (a & 63);
                        const int32_t up = p.parents[s_start[lo] + a];
                        if (up < 0 || up >= a) break;
                        a = up;
                        ++depth;
                    }
                    rope = p.lens[lo] + depth;
                }
            }
        }
        p.slots[t] = slot;
        p.positions[t] = rope;
        if (p.mask)
#pragma unroll
            for (uint32_t w = 0; w < kTreeMaxNodes / 64; ++w)
                if (w < p.n_words) p.mask[(size_t)t * p.n_words + w] = m[w];
    }
}

// ---------------------------------------------------------------------------
// paged_append
//
// (x_2i, x_2i+1) of every head turned by positions[t] * theta^(-2i/d), the
// reference's RoPE (gguf_compiler.rs:1290-1317); q to q_out, k and v to row
// slots[t] of the pools.  The angle, its sine and cosine are computed in f64
// (a far position times a frequency loses the low bits in f32) once per
// (token, pair) and shared by all heads through shared memory; the rotation
// itself is f32 (one rounding of sine and cosine, 2^-24, and one of the sum).
// Memory-bound: every value is read once and written once, 16 bytes a thread.
// ---------------------------------------------------------------------------
constexpr int kAppendThreads = 256;

template <typename T>
__device__ __forceinline__ float widen1(T x);
template <>
__device__ __forceinline__ float widen1<float>(float x) { return x; }
template <>
__device__ __forceinline__ float widen1<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float widen1<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T narrow1(float x);
template <>
__device__ __forceinline__ float narrow1<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half narrow1<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow1<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <typename T, int N>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Pack {
    T v[N];
};

template <typename S, typename Dt, int N>
__device__ __forceinline__ void turn_pack(const S *src, Dt *dst, const float2 *cs) {
    const Pack<S, N> x = *reinterpret_cast<const Pack<S, N> *>(src);
    Pack<Dt, N> y;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const float a = widen1<S>(x.v[i]), b = widen1<S>(x.v[i + 1]);
        const float2 c = cs[i / 2];
        y.v[i] = narrow1<Dt>(fmaf(a, c.x, -b * c.y));
        y.v[i + 1] = narrow1<Dt>(fmaf(a, c.y, b * c.x));
    }
    *reinterpret_cast<Pack<Dt, N> *>(dst) = y;
}

template <typename S, typename Dt, int N>
__device__ __forceinline__ void copy_pack(const S *src, Dt *dst) {
    const Pack<S, N> x = *reinterpret_cast<const Pack<S, N> *>(src);
    Pack<Dt, N> y;
#pragma unroll
    for (int i = 0; i < N; ++i) y.v[i] = narrow1<Dt>(widen1<S>(x.v[i]));
    *reinterpret_cast<Pack<Dt, N> *>(dst) = y;
}

// N elements a thread: 4 (f32 source) or 8, or 2 where a head or a pointer
// is not a multiple of 16 bytes.
template <typename S, typename Dt, int N>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const PagedAppendParams p, uint32_t tokens_at_once) {
    extern __shared__ float2 s_cs[];  // [tokens_at_once][d / 2]
    const uint32_t half = p.d / 2, nq = p.n_heads * p.d / N, nr = p.n_kv * p.d / N;
    const uint32_t per_tok = nq + 2 * nr;
    const S *q = static_cast<const S *>(p.q), *k = static_cast<const S *>(p.k), *v = static_cast<const S *>(p.v);
    S *q_out = static_cast<S *>(p.q_out);
    Dt *kp = static_cast<Dt *>(p.k_pool), *vp = static_cast<Dt *>(p.v_pool);
    const size_t row = (size_t)p.n_kv * p.d, qrow = (size_t)p.n_heads * p.d;
    for (uint32_t t0 = blockIdx.x * tokens_at_once; t0 < p.n_tokens; t0 += gridDim.x * tokens_at_once) {
        const uint32_t nt = min(tokens_at_once, p.n_tokens - t0);
        if (p.positions) {
            for (uint32_t i = threadIdx.x; i < nt * half; i += kAppendThreads) {
                const uint32_t t = i / half, j = i - t * half;
                const double freq = 1.0 / pow(p.theta, 2.0 * (double)j / (double)p.d);
                double sn, cs;
                sincos((double)p.positions[t0 + t] * freq, &sn, &cs);
                s_cs[i] = make_float2((float)cs, (float)sn);
            }
            __syncthreads();
        }
        for (uint32_t i = threadIdx.x; i < nt * per_tok; i += kAppendThreads) {
            const uint32_t t = i / per_tok;
            uint32_t e = i - t * per_tok;
            const size_t tok = t0 + t;
            const int64_t slot = p.slots[tok];
            if (slot < 0 || (uint64_t)slot >= p.n_rows) continue;
            if (e < nq) {
                const size_t at = tok * qrow + (size_t)e * N;
                if (p.positions) turn_pack<S, S, N>(q + at, q_out + at, s_cs + t * half + (e * N % p.d) / 2);
                else if (q != q_out) copy_pack<S, S, N>(q + at, q_out + at);
            } else if (e < nq + nr) {
                e -= nq;
                const size_t at = tok * row + (size_t)e * N;
                Dt *dst = kp + (size_t)slot * row + (size_t)e * N;
                if (p.positions) turn_pack<S, Dt, N>(k + at, dst, s_cs + t * half + (e * N % p.d) / 2);
                else copy_pack<S, Dt, N>(k + at, dst);
            } else {
                e -= nq + nr;
                copy_pack<S, Dt, N>(v + tok * row + (size_t)e * N, vp + (size_t)slot * row + (size_t)e * N);
            }
        }
        __syncthreads();
    }
}

bool al16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename S, typename Dt>
cudaError_t append_t(const PagedAppendParams &p, cudaStream_t st) {
    constexpr int N = sizeof(S) == 4 ? 4 : 8;
    const bool wide = p.d % 8 == 0 && al16(p.q) && al16(p.q_out) && al16(p.k) && al16(p.v) && al16(p.k_pool) && al16(p.v_pool);
    uint32_t at_once = 512 / p.d;  // about one angle a thread
    at_once = at_once < 1 ? 1 : at_once > 8 ? 8 : at_once;
    const size_t smem = p.positions ? (size_t)at_once * (p.d / 2) * sizeof(float2) : 0;
    const uint32_t blocks = (p.n_tokens + at_once - 1) / at_once, most = (uint32_t)p.num_sms * 8;
    const uint32_t grid = blocks < most ? blocks : most;
    if (wide) paged_append_kernel<S, Dt, N><<<grid, kAppendThreads, smem, st>>>(p, at_once);
    else paged_append_kernel<S, Dt, 2><<<grid, kAppendThreads, smem, st>>>(p, at_once);
    return cudaGetLastError();
}

template <typename S>
cudaError_t append_s(const PagedAppendParams &p, cudaStream_t st) {
    switch (p.dst) {
        case BML_F32: return append_t<S, float>(p, st);
        case BML_F16: return append_t<S, __half>(p, st);
        case BML_BF16: return append_t<S, __nv_bfloat16>(p, st);
    }
    return cudaErrorInvalidValue;
}

// ---------------------------------------------------------------------------
// paged_commit
//
// Row len + path[k] moves to row len + k, for k < n_accept, in the K and V of
// every layer.  path is strictly increasing (checked here: the first entry
// that is not ends the path), so path[k] >= k, and no row is written before
// it was read as long as one thread takes a column's rows in order: a later
// source path[k'] lies behind every earlier destination k < k' <= path[k'].
// One CTA per (request, layer, K or V); a thread owns one unit of the row and
// loads up to 8 rows before it stores them.
// ---------------------------------------------------------------------------
constexpr int kCommitThreads = 128;
constexpr int kCommitBatch = 8;

template <typename U>
__global__ void __launch_bounds__(kCommitThreads) paged_commit_kernel(const CommitParams p) {
    const uint32_t i = blockIdx.x, layer = blockIdx.y >> 1, which = blockIdx.y & 1;
    const int32_t len = p.lens[i], nodes = p.node_start[i + 1] - p.node_start[i];
    const int64_t room = (int64_t)p.max_pages << p.page_shift;
    int32_t want = min(p.n_accept[i], (int32_t)p.max_path);
    // a request that the plan refused, or whose rows do not fit its table, commits nothing
    if (nodes < 0 || len < 0 || p.kv_lens[i] != len + nodes || (int64_t)len + nodes > room) want = 0;
    const int32_t *path = p.path + (size_t)i * p.max_path;
    int32_t n = 0, last = -1;
    while (n < want) {
        const int32_t a = path[n];
        if (a <= last || a >= nodes) break;
        last = a;
        ++n;
    }
    if (blockIdx.y == 0 && threadIdx.x == 0) p.lens_out[i] = len + n;
    const int32_t *table = p.table + (size_t)i * p.max_pages;
    char *base = (which ? p.v_pool : p.k_pool) + (size_t)layer * p.layer_bytes;
    const uint32_t ps = 1u << p.page_shift;
    auto row_at = [&](uint32_t pos) -> char * {
        const uint32_t page = (uint32_t)table[pos >> p.page_shift];
        if (page >= p.n_pages) return nullptr;
        return base + (((size_t)page << p.page_shift) + (pos & (ps - 1))) * p.row_bytes;
    };
    for (uint32_t u = threadIdx.x; u < p.row_bytes / sizeof(U); u += kCommitThreads) {
        for (int32_t k0 = 0; k0 < n; k0 += kCommitBatch) {
            U x[kCommitBatch];
            const char *src[kCommitBatch];
#pragma unroll
            for (int b = 0; b < kCommitBatch; ++b) {
                src[b] = nullptr;
                if (k0 + b < n && path[k0 + b] != k0 + b) src[b] = row_at((uint32_t)(len + path[k0 + b]));
                if (src[b]) x[b] = reinterpret_cast<const U *>(src[b])[u];
            }
#pragma unroll
            for (int b = 0; b < kCommitBatch; ++b)
                if (src[b]) {
                    char *dst = row_at((uint32_t)(len + k0 + b));
                    if (dst) reinterpret_cast<U *>(dst)[u] = x[b];
                }
        }
    }
}

}  // namespace

cudaError_t launch_page_plan(const PlanParams &p, cudaStream_t st) {
    const size_t smem = (3 * (size_t)p.n + 1) * sizeof(int32_t);  // at most 49,156 B for kPlanMaxSeqs
    if (smem > 48 * 1024) {
        cudaError_t e = cudaFuncSetAttribute(page_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 64 * 1024);
        if (e != cudaSuccess) return e;
    }
    // a CTA takes 1024 tokens (4 a thread) or the table entries of 32 requests, whichever asks for more CTAs
    const uint32_t by_tok = (p.n_tokens + 1023) / 1024, by_seq = (p.n + 31) / 32;
    uint32_t grid = by_tok > by_seq ? by_tok : by_seq;
    grid = grid < 1 ? 1 : grid > (uint32_t)p.num_sms * 4 ? (uint32_t)p.num_sms * 4 : grid;
    page_plan_kernel<<<grid, kPlanThreads, smem, st>>>(p);
    return cudaGetLastError();
}

cudaError_t launch_paged_append(const PagedAppendParams &p, cudaStream_t st) {
    if (p.n_tokens == 0) return cudaSuccess;
    switch (p.src) {
        case BML_F32: return append_s<float>(p, st);
        case BML_F16: return append_s<__half>(p, st);
        case BML_BF16: return append_s<__nv_bfloat16>(p, st);
    }
    return cudaErrorInvalidValue;
}

cudaError_t launch_paged_commit(const CommitParams &p, cudaStream_t st) {
    const dim3 grid(p.n, p.n_layers * 2);
    const bool a16 = p.row_bytes % 16 == 0 && al16(p.k_pool) && al16(p.v_pool) && p.layer_bytes % 16 == 0;
    if (a16) paged_commit_kernel<uint4><<<grid, kCommitThreads, 0, st>>>(p);
    else paged_commit_kernel<uint16_t><<<grid, kCommitThreads, 0, st>>>(p);
    return cudaGetLastError();
}

}  // namespace bml
