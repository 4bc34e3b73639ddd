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
// Block-wide exclusive scan of two 64-bit values per thread
// ---------------------------------------------------------------------------
struct Pair64 {
    int64_t x, y;
};
__device__ __forceinline__ Pair64 block_scan(Pair64 v, Pair64 *warp_sums, Pair64 *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    Pair64 inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t a = __shfl_up_sync(0xffffffffu, inc.x, o), b = __shfl_up_sync(0xffffffffu, inc.y, o);
        if (lane >= o) {
            inc.x += a;
            inc.y += b;
        }
    }
    if (lane == 31) warp_sums[warp] = inc;
    __syncthreads();
    Pair64 before = {0, 0}, all = {0, 0};
    for (int w = 0; w < nw; ++w) {
        const Pair64 s = warp_sums[w];
        if (w < warp) {
            before.x += s.x;
            before.y += s.y;
        }
        all.x += s.x;
        all.y += s.y;
    }
    __syncthreads();
    *total = all;
    return {before.x + inc.x - v.x, before.y + inc.y - v.y};
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

// kRun: consecutive tokens of a thread.  4 without drafts, where they mostly
// share a request and a page (no parents then); 1 with drafts, whose threads
// walk a tree each (16 drafts, 500 tokens took 1.6 times as long with 4).
template <uint32_t kRun>
__global__ void __launch_bounds__(kPlanThreads) page_plan_kernel(const PlanParams p) {
    extern __shared__ int32_t sh[];
    int32_t *s_start = sh;                 // [n + 1] first token
    int32_t *s_base = sh + p.n + 1;        // [n] first new page's place in the free list
    int32_t *s_own = s_base + p.n;         // [n] pages held before, or -1: refused
    __shared__ Pair64 warp_sums[kPlanThreads / 32];
    const uint32_t per = (p.n + kPlanThreads - 1) / kPlanThreads;
    const uint32_t i0 = min(threadIdx.x * per, p.n), i1 = min(i0 + per, p.n);
    const int64_t ps = 1ll << p.page_shift;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int32_t used_now = *p.free_used;  // on its way with the lengths

    // A request that is bad takes no pages, and neither does one whose tokens do
    // not fit: that is known only after the scan of the tokens, so in the rare
    // case that they do not all fit the pages are summed again.
    auto verify = [&](uint32_t i, int64_t end, int64_t &add) {
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
    Pair64 mine = {0, 0}, all;
    for (uint32_t i = i0; i < i1; ++i) {
        int64_t add;
        verify(i, 0, add);
        mine.x += max(p.n_new[i], 0);
        mine.y += add;
    }
    Pair64 before = block_scan(mine, warp_sums, &all);
    const int64_t first_tok = before.x, all_tok = all.x;
    int64_t at = first_tok;
    if (all_tok > p.n_tokens) {
        mine.y = 0;
        for (uint32_t i = i0; i < i1; ++i) {
            int64_t add;
            at += max(p.n_new[i], 0);
            verify(i, at, add);
            mine.y += add;
        }
        before = block_scan(mine, warp_sums, &all);
    }
    int64_t cum = before.y;
    const int64_t used = min(max(used_now, 0), (int32_t)p.n_free);
    const int64_t avail = (int64_t)p.n_free - used;
    int64_t granted = 0;  // largest running sum that still fits
    at = first_tok;
    for (uint32_t i = i0; i < i1; ++i) {
        int64_t add;
        const int64_t begin = at;
        at += max(p.n_new[i], 0);
        int32_t st = verify(i, at, add);
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
        if ((threadIdx.x & 31) == 0) warp_sums[threadIdx.x >> 5].x = granted;
    }
    __syncthreads();
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        p.node_start[p.n] = s_start[p.n];
        int64_t g = 0;
        for (int w = 0; w < kPlanThreads / 32; ++w) g = g > warp_sums[w].x ? g : warp_sums[w].x;
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
    const uint32_t runs = (p.n_tokens + kRun - 1) / kRun;
    const bool wide = ((reinterpret_cast<uintptr_t>(p.slots) | reinterpret_cast<uintptr_t>(p.positions)) & 15u) == 0;
    for (uint32_t run = blockIdx.x * kPlanThreads + threadIdx.x; run < runs; run += gridDim.x * kPlanThreads) {
        const uint32_t first = run * kRun;
        int64_t slot[kRun];
        int32_t rope[kRun];
        uint32_t lo = 0;
        if ((int32_t)first < total) {
            // the last request that starts at or before it (empty ones in between have the same start)
            uint32_t hi = p.n;
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) >> 1;
                if (s_start[mid] <= (int32_t)first) lo = mid;
                else hi = mid;
            }
        }
        int32_t own = s_own[lo];
        int64_t len = p.lens[lo], held = -1, page = 0;  // page: of index held in the request's table
        const int32_t j0 = (int32_t)first - s_start[lo];
        if (kRun == 4 && own >= 0 && j0 >= 0 && (int32_t)first + 4 <= s_start[lo + 1]) {
            // tokens of one request, on one page or two (1.05 M tokens of 512
            // requests 11.8 -> 9.1 us)
            auto page_of = [&](uint32_t pg) -> int64_t {
                return (int64_t)(pg < (uint32_t)own ? p.table[(size_t)lo * p.max_pages + pg] : p.free_pages[s_base[lo] + (pg - own)])
                       << p.page_shift;
            };
            const uint32_t pos = (uint32_t)len + j0, off = pos & ((uint32_t)ps - 1), pg = pos >> p.page_shift;
            const int64_t a = page_of(pg) + off, b = off + 3 < (uint32_t)ps ? a : page_of(pg + 1) + off - ps;
#pragma unroll
            for (uint32_t u = 0; u < kRun; ++u) {
                slot[u] = (off + u < (uint32_t)ps ? a : b) + u;
                rope[u] = (int32_t)(pos + u);
            }
        } else {
#pragma unroll
            for (uint32_t u = 0; u < kRun; ++u) {
                const int32_t t = (int32_t)(first + u);
                slot[u] = -1;
                rope[u] = 0;
                uint64_t m[kTreeMaxNodes / 64] = {0, 0, 0, 0};
                if (t < total) {
                    if (t >= s_start[lo + 1]) {
                        do ++lo;
                        while (t >= s_start[lo + 1]);
                        own = s_own[lo];
                        len = p.lens[lo];
                        held = -1;
                    }
                    if (own >= 0) {
                        const int32_t j = t - s_start[lo];
                        const int64_t pos = len + j, pg = pos >> p.page_shift;
                        if (pg != held) {
                            page = pg < own ? p.table[(size_t)lo * p.max_pages + pg] : p.free_pages[s_base[lo] + (pg - own)];
                            held = pg;
                        }
                        slot[u] = (page << p.page_shift) + (pos & (ps - 1));
                        rope[u] = (int32_t)pos;
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
                            rope[u] = (int32_t)len + depth;
                        }
                    }
                }
                if (p.mask && first + u < p.n_tokens)
#pragma unroll
                    for (uint32_t w = 0; w < kTreeMaxNodes / 64; ++w)
                        if (w < p.n_words) p.mask[(size_t)t * p.n_words + w] = m[w];
            }
        }
        if (kRun == 4 && wide && first + kRun <= p.n_tokens) {
            longlong2 *s2 = reinterpret_cast<longlong2 *>(p.slots + first);
            s2[0] = make_longlong2(slot[0], slot[1 % kRun]);
            s2[1] = make_longlong2(slot[2 % kRun], slot[3 % kRun]);
            *reinterpret_cast<int4 *>(p.positions + first) = make_int4(rope[0], rope[1 % kRun], rope[2 % kRun], rope[3 % kRun]);
        } else {
#pragma unroll
            for (uint32_t u = 0; u < kRun; ++u)
                if (first + u < p.n_tokens) {
                    p.slots[first + u] = slot[u];
                    p.positions[first + u] = rope[u];
                }
        }
    }
}

// ---------------------------------------------------------------------------
// paged_append
//
// (x_2i, x_2i+1) of every head turned by positions[t] * theta^(-2i/d), the
// reference's RoPE (gguf_compiler.rs:1290-1317); q to q_out, k and v to row
// slots[t] of the pools.  Angle, sine and cosine are computed in f64 (a far
// position times a frequency loses the low bits in f32) once per (token, pair)
// and shared by all heads through shared memory; the rotation itself is f32
// (one rounding of sine and cosine, 2^-24, and one of the sum).
// Memory-bound: every value is read once and written once, 16 bytes a thread,
// a thread's pieces of kAtOnce tokens in flight together.
// ---------------------------------------------------------------------------
constexpr int kAppendThreads = 256;
constexpr int kAtOnce = 4;

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

// Streaming loads and stores: 16,001 tokens of 32 + 8 + 8 heads of 128 bf16 in
// 77 us (5.1 TB/s), 81 without.
template <typename S, int N>
__device__ __forceinline__ Pack<S, N> load_pack(const S *src) {
    if (sizeof(Pack<S, N>) == 16) {
        const uint4 z = __ldcs(reinterpret_cast<const uint4 *>(src));
        return *reinterpret_cast<const Pack<S, N> *>(&z);
    }
    return *reinterpret_cast<const Pack<S, N> *>(src);
}

// x turned by cs (cosine, sine) per pair, or as is
template <typename S, typename Dt, int N>
__device__ __forceinline__ void put_pack(const Pack<S, N> &x, Dt *dst, const float2 *cs) {
    Pack<Dt, N> y;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const float a = widen1<S>(x.v[i]), b = widen1<S>(x.v[i + 1]);
        if (cs) {
            const float2 c = cs[i / 2];
            y.v[i] = narrow1<Dt>(fmaf(a, c.x, -b * c.y));
            y.v[i + 1] = narrow1<Dt>(fmaf(a, c.y, b * c.x));
        } else {
            y.v[i] = narrow1<Dt>(a);
            y.v[i + 1] = narrow1<Dt>(b);
        }
    }
    if (sizeof(y) == 16) __stcs(reinterpret_cast<uint4 *>(dst), *reinterpret_cast<const uint4 *>(&y));
    else *reinterpret_cast<Pack<Dt, N> *>(dst) = y;
}

// (cos x, sin x) for x >= 0 from f64: x = k pi/2 + r with |r| <= pi/4 (pi/2 as
// the sum of two f64), the Taylor series of sine to r^9 and of cosine to r^10
// (remainders below 2e-9), and the quadrant.  About 20 f64 operations.
__device__ __forceinline__ float2 cos_sin(double x) {
    const double k = rint(x * 0.63661977236758134308);
    double r = fma(-k, 1.57079632679489661923, x);
    r = fma(-k, 6.12323399573676603587e-17, r);
    const double z = r * r;
    double s = fma(z, 1.0 / 362880.0, -1.0 / 5040.0);
    s = fma(z, s, 1.0 / 120.0);
    s = fma(z, s, -1.0 / 6.0);
    s = fma(r * z, s, r);
    double c = fma(z, -1.0 / 3628800.0, 1.0 / 40320.0);
    c = fma(z, c, -1.0 / 720.0);
    c = fma(z, c, 1.0 / 24.0);
    c = fma(z, c, -0.5);
    c = fma(z, c, 1.0);
    const int q = (int)((long long)k & 3);
    const float fs = (float)s, fc = (float)c;
    const float a = (q & 1) ? fs : fc, b = (q & 1) ? fc : fs;
    return make_float2((q == 1 || q == 2) ? -a : a, q >= 2 ? -b : b);
}

// N elements a thread: 4 (f32 source) or 8, or 2 where a head or a pointer
// is not a multiple of 16 bytes.
template <typename S, typename Dt, int N>
__global__ void __launch_bounds__(kAppendThreads, 4) paged_append_kernel(const PagedAppendParams p, uint32_t at_once) {
    extern __shared__ float2 s_cs[];  // [at_once][d / 2]
    const uint32_t half = p.d / 2, per_head = p.d / N, nq = p.n_heads * per_head, nr = p.n_kv * per_head;
    const S *q = static_cast<const S *>(p.q), *k = static_cast<const S *>(p.k), *v = static_cast<const S *>(p.v);
    S *q_out = static_cast<S *>(p.q_out);
    Dt *kp = static_cast<Dt *>(p.k_pool), *vp = static_cast<Dt *>(p.v_pool);
    const size_t row = (size_t)p.n_kv * p.d, qrow = (size_t)p.n_heads * p.d;
    // a thread's pair stays the same where half divides the thread count
    const bool fixed = kAppendThreads % half == 0;
    double freq = fixed ? exp2(-2.0 * (double)(threadIdx.x % half) / (double)p.d * p.log2_theta) : 0.0;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t g0 = blockIdx.x * at_once, nt = min(at_once, p.n_tokens - g0);
    if (p.positions) {
        for (uint32_t i = threadIdx.x; i < nt * half; i += kAppendThreads) {
            const uint32_t t = i / half;
            if (!fixed) freq = exp2(-2.0 * (double)(i - t * half) / (double)p.d * p.log2_theta);
            s_cs[i] = cos_sin((double)max(p.positions[g0 + t], 0) * freq);
        }
        __syncthreads();
    }
    for (uint32_t e0 = threadIdx.x; e0 < nq + 2 * nr; e0 += kAppendThreads) {
        // which array, and where in a token's row of it
        const int what = e0 < nq ? 0 : e0 < nq + nr ? 1 : 2;
        const uint32_t e = e0 - (what == 0 ? 0 : what == 1 ? nq : nq + nr);
        const S *src = (what == 0 ? q : what == 1 ? k : v) + (size_t)e * N;
        const size_t stride = what == 0 ? qrow : row;
        const float2 *cs = what < 2 && p.positions ? s_cs + e % per_head * (N / 2) : nullptr;
        if (what == 0 && !cs && q == q_out) continue;
        for (uint32_t t0 = 0; t0 < nt; t0 += kAtOnce) {
            Pack<S, N> x[kAtOnce];
            int64_t slot[kAtOnce];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const uint32_t t = t0 + u;
                slot[u] = t < nt ? p.slots[g0 + t] : -1;
                if (t < nt) x[u] = load_pack<S, N>(src + (size_t)(g0 + t) * stride);
            }
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                if (slot[u] < 0 || (uint64_t)slot[u] >= p.n_rows) continue;
                const float2 *c = cs ? cs + (t0 + u) * half : nullptr;
                if (what == 0) put_pack<S, S, N>(x[u], q_out + (size_t)(g0 + t0 + u) * qrow + (size_t)e * N, c);
                else put_pack<S, Dt, N>(x[u], (what == 1 ? kp : vp) + (size_t)slot[u] * row + (size_t)e * N, c);
            }
        }
    }
}

bool al16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename S, typename Dt>
cudaError_t append_t(const PagedAppendParams &p, cudaStream_t st) {
    constexpr int N = sizeof(S) == 4 ? 4 : 8;
    const bool wide = p.d % 8 == 0 && al16(p.q) && al16(p.q_out) && al16(p.k) && al16(p.v) && al16(p.k_pool) && al16(p.v_pool);
    // tokens of a CTA at a time: about one angle a thread, but every SM has one first
    uint32_t at_once = 512 / p.d, spread = p.n_tokens / p.num_sms;
    at_once = at_once > spread ? spread : at_once;
    at_once = at_once < 1 ? 1 : at_once > 8 ? 8 : at_once;
    const size_t smem = p.positions ? (size_t)at_once * (p.d / 2) * sizeof(float2) : 0;
    const uint32_t grid = (p.n_tokens + at_once - 1) / at_once;  // more CTAs than fit: the hardware balances them
    return wide ? launch_after(paged_append_kernel<S, Dt, N>, dim3(grid), kAppendThreads, (int)smem, st, p, at_once)
                : launch_after(paged_append_kernel<S, Dt, 2>, dim3(grid), kAppendThreads, (int)smem, st, p, at_once);
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
    asm volatile("griddepcontrol.wait;" ::: "memory");
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
    auto kern = p.parents ? page_plan_kernel<1> : page_plan_kernel<4>;
    // without the allowance the dynamic and the static part (warp_sums) together have 48 KB
    if (smem + kPlanThreads / 32 * sizeof(Pair64) > 48 * 1024) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 64 * 1024);
        if (e != cudaSuccess) return e;
    }
    // a CTA takes 1024 tokens (4 a thread; of drafts 256) or the table entries of 32
    // requests, whichever asks for more CTAs
    const uint32_t each = p.parents ? 256 : 1024;
    const uint32_t by_tok = (p.n_tokens + each - 1) / each, by_seq = (p.n + 31) / 32;
    uint32_t grid = by_tok > by_seq ? by_tok : by_seq;
    grid = grid < 1 ? 1 : grid > (uint32_t)p.num_sms * 2 ? (uint32_t)p.num_sms * 2 : grid;
    return launch_after(kern, dim3(grid), kPlanThreads, (int)smem, st, p);
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
    return a16 ? launch_after(paged_commit_kernel<uint4>, grid, kCommitThreads, 0, st, p)
               : launch_after(paged_commit_kernel<uint16_t>, grid, kCommitThreads, 0, st, p);
}

}  // namespace bml
