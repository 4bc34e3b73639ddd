// tree_umma32.cu -- attention of drafted tokens over a paged cache of 32-bit
// values on tcgen05 tensor cores (sm_100a): results to about f32 precision
// from TF32 products.
//
// The mathematics and the schedule are those of tree.cu / tree.cuh: a CTA (one
// per SM) works through its even share of the line of 64-position tiles,
// segment by segment.  A unit is one request, kv head and group of up to RT
// query rows, RT = the most whole tokens' rows that fit 128; row r of it is
// (node r / group, q head r % group) and TMEM lane r.
//
// Every f32 operand x is hi + lo with hi = x rounded to TF32 and lo = x - hi,
// of which the tensor core takes the upper bits (22 together), and a product is
// hi*hi + (lo*hi + hi*lo).  The tensor core's sums truncate, so S's two parts
// are summed apart, and a tile's O (its small terms first) is added to the
// output in registers, with a rounding, and not summed on from tile to tile in
// tensor memory.
//
//   Q hi, lo     tensor memory (D columns each), written once a segment;
//   K hi, lo     shared memory, K-major as it arrives; hi replaces K, lo is the
//                next 64 rows of the MMA's B operand;
//   P hi, lo     tensor memory, hi over S;
//   V hi, lo     shared memory, transposed on the way (positions are the MMA's
//                K index).
//
//   warp 0       copies K and V tiles (cp.async.bulk.tensor; K two stages)
//   warp 1       tensor memory, and every tcgen05.mma
//   warps 2-9    thread = row = TMEM lane and half of the columns: Q; the
//                softmax (the halves' maxima meet in shared memory); O added
//                in registers; the rows written
//   warps 10-15  split K and V.
//
// V is split while S is computed, and the next tile's K after it.
//
// Measured on B200, d = 128: 3.55 us a tile and CTA, of which the S products
// take 1.6 (1.0 while nothing else uses shared memory), the softmax 1.4 and P V
// 0.9, one after another: Q's two parts, S and O fill the tensor memory, so S
// has no second buffer; copies, splits and MMA operands pass 3600 cycles' worth
// of shared memory.  4 requests of 618 to 2671 positions, 32 to 84 rows: 43 us,
// 75.6 with tree.cu's kernel.
//
// What a row does not see must not reach it: scores are replaced by -inf (bad
// pages, rows past the length, nodes outside the mask), V rows past the length
// and values of drafted nodes that are not finite are split as zeros, and
// tree_nonfinite adds the latter to the rows that see them.
#include <math.h>

#include "tree.cuh"
#include "umma.cuh"

namespace bml {

namespace {

constexpr int BM = 128, BN = 64;
constexpr int kRowWarps = 8, kSplitWarps = 6;
constexpr int kThreads = 32 * (2 + kRowWarps + kSplitWarps);  // 512: up to 128 registers a thread
constexpr int kBadRing = 16;  // tiles whose page flags are kept

template <int D>
struct XCfg {
    static constexpr int KB = D / 32;          // 128-byte column blocks of a K row
    static constexpr int TILE = BN * D * 4;    // a K or V tile
    static constexpr int OFF_K = 0;            // two stages: per column block 64 rows hi (in place), 64 rows lo
    static constexpr int OFF_V = 4 * TILE;
    static constexpr int OFF_VHI = 5 * TILE;   // [2 blocks of 32 positions][D][128 B]
    static constexpr int OFF_VLO = 6 * TILE;
    static constexpr int OFF_SH = 7 * TILE;
    static constexpr int SMEM = OFF_SH + 3 * 1024;
    // tensor memory columns
    static constexpr uint32_t QHI = 0, QLO = D, OC = 2 * D;
    static constexpr uint32_t SC = 3 * D, PLO = SC + BN;  // S: Q hi * K hi, and the other two products; then P
    static constexpr uint32_t TMEM_COLS = 512;
};
static_assert(XCfg<128>::SMEM <= 227 * 1024 && XCfg<128>::PLO + BN == 512, "shared and tensor memory");

struct XParams {
    CUtensorMap tk, tv;  // (d, n_kv, rows); box (32, 1, box_rows) swizzled, (d, 1, box_rows) plain
    TreeParams t;
    uint32_t box_rows;  // min(page, 64)
};

struct alignas(16) XShared {
    uint64_t k_full[2], k_empty[2], k_ready[2];
    uint64_t v_full, v_empty, q_ready, v_ready, s_full, p_ready, o_full, o_free, drain;
    uint32_t tmem, abort;
    uint32_t bad[kBadRing];  // per tile: 16-position blocks on pages outside the pool
    uint32_t odd[3];  // [segment % 3]: the last segment (from 1 on) with a drafted node's V value that is not finite
    float top[2][BM], sum[2][BM];  // [half][row]: maximum of a tile; l of a segment
    TreeShared sched;
};
static_assert(sizeof(XShared) <= 3 * 1024, "small arrays");

// D[tmem] (+)= A[tmem] * B[smem desc], TF32: A is M x 8, 8 columns.
__device__ __forceinline__ void mma_tf32_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::tf32 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// 32 values as hi and lo, to tensor memory.  kAny: of any size (else weights).
template <bool kAny>
__device__ __forceinline__ void put_split(uint32_t hi_at, uint32_t lo_at, const float *x) {
#pragma unroll
    for (int c = 0; c < 32; c += 16) {
        uint32_t hi[16], lo[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            if (kAny) tf32_split_any(x[c + k], hi[k], lo[k]);
            else tf32_split(x[c + k], hi[k], lo[k]);
        }
        tmem_st16(hi_at + c, hi);
        tmem_st16(lo_at + c, lo);
    }
}

// Which of the 32 positions from node0 on (negative: committed ones, seen by
// all) node t sees.
__device__ __forceinline__ uint32_t see_half(const TreeParams &p, const TreeSeq &s, uint32_t t, int32_t node0) {
    if (s.L == 0) return 0u;
    uint32_t see = 0;
#pragma unroll 1
    for (int b = 0; b < 2; ++b) {
        const int32_t n0 = node0 + 16 * b;
        see |= (n0 <= -16 ? 0xffffu : tree_see16(p, s, t, n0) & 0xffffu) << (16 * b);
    }
    return see;
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1) tree_umma32_kernel(const __grid_constant__ XParams xp) {
    using C = XCfg<D>;
    const TreeParams &p = xp.t;
    extern __shared__ __align__(1024) uint8_t smem[];
    XShared &sh = *reinterpret_cast<XShared *>(smem + C::OFF_SH);
    volatile uint32_t *abort_flag = &sh.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.k_full[i], 1);
            mbar_init(&sh.k_empty[i], 1);
            mbar_init(&sh.k_ready[i], kSplitWarps);
        }
        mbar_init(&sh.v_full, 1);
        mbar_init(&sh.v_empty, kSplitWarps);
        mbar_init(&sh.q_ready, kRowWarps);
        mbar_init(&sh.v_ready, kSplitWarps);
        mbar_init(&sh.s_full, 1);
        mbar_init(&sh.p_ready, kRowWarps);
        mbar_init(&sh.o_full, 1);
        mbar_init(&sh.o_free, kRowWarps);
        mbar_init(&sh.drain, 1);
        sh.abort = 0u;
        fence_mbar_init();
    }
    if (threadIdx.x < 3) sh.odd[threadIdx.x] = 0u;
    if (warp == 0 && lane == 0) {
        prefetch_tmap(&xp.tk);
        prefetch_tmap(&xp.tv);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)),
                     "r"(C::TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const TreeRange range = tree_range<false>(p, &sh.sched, blockIdx.x, gridDim.x);
    __syncthreads();  // the set-up above
    tc_fence_after();
    const uint32_t tmem = *(volatile uint32_t *)&sh.tmem;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the merge, which waits for this grid
    TreeWalk<false> walk(range);
    TreeSeg sg = {};
    uint32_t it = 0, segs = 0;  // tiles, segments so far

    if (warp == 0) {
        // --------------------------------------------------------------- producer
        // Lanes 0-15 issue K's boxes (column block lane % KB of part lane / KB),
        // lanes 16-19 V's (part lane - 16).
        const uint64_t policy = l2_policy_evict_first();
        const uint32_t parts = BN / xp.box_rows, ps_mask = (1u << p.page_shift) - 1;
        const bool is_k = lane < 16;
        const uint32_t part = is_k ? lane / C::KB : lane - 16, kb = is_k ? lane % C::KB : 0u;
        const bool mine = part < parts && lane < 20;
        bool live = !(p.diag & kTreeStall);
        while (live && walk.next(p, sg)) {
            const int32_t *table = p.table + (size_t)sg.seq * p.max_pages;
            // a lane's first row in the pool of tile j (-1: past the length, -2: a page outside the pool)
            auto row_of = [&](uint32_t j) -> int {
                const uint32_t pos = j * BN + part * xp.box_rows;
                if (!mine || pos >= sg.s.L) return -1;
                const uint32_t page = (uint32_t)table[pos >> p.page_shift];
                return page < p.n_pages ? (int)((page << p.page_shift) + (pos & ps_mask)) : -2;
            };
            int next = row_of(sg.t0);
            for (uint32_t j = sg.t0; j < sg.t1; ++j, ++it) {
                const int row = next;
                if (j + 1 < sg.t1) next = row_of(j + 1);
                const uint32_t st = it & 1u, use = it >> 1;
                const uint32_t bits = xp.box_rows / 16;
                uint32_t flag = 0;
                if (__any_sync(0xffffffffu, row == -2))
                    flag = __reduce_or_sync(0xffffffffu, row == -2 ? ((1u << bits) - 1) << (part * bits) : 0u);
                if (lane == 0) *(volatile uint32_t *)&sh.bad[it % kBadRing] = flag;
                // a page outside the pool is read past the map's end: zeros
                const int at = row == -2 ? (int)(p.n_pages << p.page_shift) : row;
                const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, row != -1 && !is_k)) * xp.box_rows * D * 4;
                const bool once = sg.s.groups == 1;  // K and V are read once
                auto copy = [&](bool k, uint64_t *full, uint8_t *dst) {
                    if (lane == 0) mbar_arrive_expect_tx(full, bytes);
                    __syncwarp();
                    if (row != -1 && is_k == k) {
                        if (once) tma_load_3d_hint(dst, k ? &xp.tk : &xp.tv, (int)kb * 32, (int)sg.head, at, full, policy);
                        else tma_load_3d(dst, k ? &xp.tk : &xp.tv, (int)kb * 32, (int)sg.head, at, full);
                    }
                    __syncwarp();
                };
                if (use > 0) live = __all_sync(0xffffffffu, wait_bar(&sh.k_empty[st], (use & 1u) ^ 1u, abort_flag, p.wait_ns));
                if (!live) break;
                copy(true, &sh.k_full[st], smem + C::OFF_K + st * 2 * C::TILE + kb * 2 * BN * 128 + part * xp.box_rows * 128);
                if (it > 0) live = __all_sync(0xffffffffu, wait_bar(&sh.v_empty, (it & 1u) ^ 1u, abort_flag, p.wait_ns));
                if (!live) break;
                copy(false, &sh.v_full, smem + C::OFF_V + part * xp.box_rows * D * 4);
            }
        }
        // No copy may outlive the CTA: all have landed unless a wait gave up,
        // and then none is issued any more, so those that have not will soon.
        if (!live) {
            const uint64_t t0 = globaltimer_ns();
            while (globaltimer_ns() - t0 < 1000000ull) {}
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------------------- MMA issuer
        // 2: TF32.  Q hi meets K hi and lo in one MMA of 128 columns (an MMA of 64
        // takes as long), Q lo only K hi.
        constexpr uint32_t idesc_qk = make_idesc(2u, BM, 2 * BN, 0), idesc_lo = make_idesc(2u, BM, BN, 0), idesc_pv = make_idesc(2u, BM, D, 0);
        const uint64_t d_k = smem_desc(smem_u32(smem + C::OFF_K), 16, 1024);
        const uint64_t d_vhi = smem_desc(smem_u32(smem + C::OFF_VHI), 16, 1024), d_vlo = smem_desc(smem_u32(smem + C::OFF_VLO), 16, 1024);
        bool live = true;
        auto wait_all = [&](uint64_t *bar, uint32_t parity) {
            live = live && __all_sync(0xffffffffu, wait_bar(bar, parity, abort_flag, p.wait_ns));
            __syncwarp();
            tc_fence_after();
        };
        // one term's chain over kK columns of A
        auto chain = [&](uint32_t d, uint32_t a, uint64_t b, uint32_t block, uint32_t idesc, int n, bool first) {
            for (int kk = 0; kk < n; ++kk) {
                const uint32_t off = ((kk >> 2) * block + (kk & 3) * 32) >> 4;
                if (elect_one()) mma_tf32_ts(d, a + kk * 8, b + off, idesc, first && kk == 0 ? 0u : 1u);
                __syncwarp();
            }
        };
        while (live && walk.next(p, sg)) {
            wait_all(&sh.q_ready, segs & 1u);
            for (uint32_t j = sg.t0; j < sg.t1 && live; ++j, ++it) {
                const uint32_t st = it & 1u, par = it & 1u;
                wait_all(&sh.k_ready[st], (it >> 1) & 1u);
                if (!live) break;
                const uint64_t k = d_k + ((st * 2 * C::TILE) >> 4);
                chain(tmem + C::SC, tmem + C::QHI, k, 2 * BN * 128, idesc_qk, D / 8, true);
                chain(tmem + C::PLO, tmem + C::QLO, k, 2 * BN * 128, idesc_lo, D / 8, false);
                if (elect_one()) {
                    tc_commit(&sh.s_full);
                    tc_commit(&sh.k_empty[st]);
                }
                __syncwarp();
                wait_all(&sh.v_ready, par);
                if (it > 0) wait_all(&sh.o_free, par ^ 1u);
                wait_all(&sh.p_ready, par);
                if (!live) break;
                chain(tmem + C::OC, tmem + C::PLO, d_vhi, D * 128, idesc_pv, BN / 8, true);
                chain(tmem + C::OC, tmem + C::SC, d_vlo, D * 128, idesc_pv, BN / 8, false);
                chain(tmem + C::OC, tmem + C::SC, d_vhi, D * 128, idesc_pv, BN / 8, false);
                if (elect_one()) tc_commit(&sh.o_full);
                __syncwarp();
            }
            ++segs;
        }
        if (elect_one()) tc_commit(&sh.drain);  // no MMA outlives the CTA
        __syncwarp();
        mbar_drain(&sh.drain, 0, p.wait_ns);
        __syncwarp();
    } else if (warp < 2 + kRowWarps) {
        // ---------------------------------------------------------- Q and softmax
        const uint32_t q4 = warp & 3, half = (warp - 2) >> 2, r = q4 * 32 + lane;
        const uint32_t at = tmem + ((q4 * 32) << 16), hi_at = at + C::SC + 32 * half, lo_at = at + C::PLO + 32 * half, o_at = at + C::OC + half * (D / 2);
        while (walk.next(p, sg)) {
            const bool valid = r < sg.rows;
            const bool warp_live = q4 * 32 < sg.rows;
            const uint32_t P = sg.s.L - min(sg.s.T, sg.s.L), t = min((sg.row0 + r) / p.group, sg.s.T - 1);
            if (warp_live) {
                const float *q = static_cast<const float *>(p.q) + (valid ? tree_row(p, sg, sg.row0 + r, D) : 0);
                float x[D / 2];
#pragma unroll
                for (int u = 0; u < D / 8; ++u) {
                    const float4 y = valid ? *reinterpret_cast<const float4 *>(q + half * (D / 2) + 4 * u) : make_float4(0.f, 0.f, 0.f, 0.f);
                    x[4 * u] = y.x;
                    x[4 * u + 1] = y.y;
                    x[4 * u + 2] = y.z;
                    x[4 * u + 3] = y.w;
                }
                __syncwarp();
#pragma unroll
                for (int c = 0; c < D / 2; c += 32) put_split<true>(at + C::QHI + half * (D / 2) + c, at + C::QLO + half * (D / 2) + c, x + c);
                tmem_wait_st();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.q_ready);
            float m = -INFINITY, l = 0.f;  // l: of this half of the positions
            float o[D / 2];                // this half of the columns
#pragma unroll
            for (int k = 0; k < D / 2; ++k) o[k] = 0.f;
            for (uint32_t j = sg.t0; j < sg.t1; ++j, ++it) {
                wait_bar(&sh.s_full, it & 1u, abort_flag, p.wait_ns);
                __syncwarp();
                tc_fence_after();
                float alpha = 1.f;
                if (warp_live) {
                    const uint32_t bad = *(volatile uint32_t *)&sh.bad[it % kBadRing] >> (2 * half) & 3u, kv0 = j * BN + 32 * half;
                    const bool edge = kv0 + 32 > P;
                    uint32_t see = ~0u;
                    if (edge || bad) {
                        if (edge) see = see_half(p, sg.s, t, (int32_t)(kv0 - P));
                        if (bad & 1) see &= 0xffff0000u;
                        if (bad & 2) see &= 0x0000ffffu;
                    }
                    float s[32];
                    tmem_ld32(hi_at, s);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float y[16];
                        tmem_ld16(lo_at + 16 * h, y);
                        tmem_wait_ld();
#pragma unroll
                        for (int k = 0; k < 16; k += 2) {
                            const float2 z = __fadd2_rn(make_float2(s[16 * h + k], s[16 * h + k + 1]), make_float2(y[k], y[k + 1]));
                            s[16 * h + k] = z.x;
                            s[16 * h + k + 1] = z.y;
                        }
                    }
                    if (edge || bad) {
#pragma unroll
                        for (int k = 0; k < 32; ++k)
                            if (!(see >> k & 1)) s[k] = -INFINITY;
                    }
                    float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                    for (int k = 4; k < 32; ++k) mx[k & 3] = fmaxf(mx[k & 3], s[k]);
                    const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale_log2;  // > 0
                    sh.top[half][r] = top;
                    named_bar_sync(2 + q4, 64);
                    const float m_new = fmaxf(m, fmaxf(top, sh.top[half ^ 1u][r]));
                    const float mu = m_new == -INFINITY ? 0.f : m_new;
                    alpha = fast_exp2(m - mu);
                    m = m_new;
                    const float2 c2 = make_float2(p.scale_log2, p.scale_log2), nm2 = make_float2(-mu, -mu);
                    float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                    for (int k = 0; k < 32; k += 2) {
                        const float2 z = __ffma2_rn(make_float2(s[k], s[k + 1]), c2, nm2);
                        s[k] = fast_exp2(z.x);
                        s[k + 1] = fast_exp2(z.y);
                        sum[k >> 1 & 1] = __fadd2_rn(sum[k >> 1 & 1], make_float2(s[k], s[k + 1]));
                    }
                    put_split<false>(hi_at, lo_at, s);
                    const float2 both = __fadd2_rn(sum[0], sum[1]);
                    l = fmaf(l, alpha, both.x + both.y);
                    tmem_wait_st();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.p_ready);
                wait_bar(&sh.o_full, it & 1u, abort_flag, p.wait_ns);
                __syncwarp();
                tc_fence_after();
                if (warp_live)
#pragma unroll
                    for (int c = 0; c < D / 2; c += 16) {
                        float y[16];
                        tmem_ld16(o_at + c, y);
                        tmem_wait_ld();
#pragma unroll
                        for (int u = 0; u < 16; u += 2) {
                            const float2 z = __ffma2_rn(make_float2(o[c + u], o[c + u + 1]), make_float2(alpha, alpha), make_float2(y[u], y[u + 1]));
                            o[c + u] = z.x;
                            o[c + u + 1] = z.y;
                        }
                    }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.o_free);
            }
            if (warp_live) {
                sh.sum[half][r] = l;
                named_bar_sync(2 + q4, 64);
                l += sh.sum[half ^ 1u][r];
            }
            if (*abort_flag) l = __int_as_float(0x7fffffff);  // a wait gave up: NaN
            const float inv = l == 0.f ? 0.f : 1.f / l;
            // all V of the segment has been split
            const bool odd = sg.t1 * BN > P && *(const volatile uint32_t *)&sh.odd[segs % 3] == segs + 1;
            float *part = sg.slot < 2 ? tree_part(p, D, blockIdx.x, sg.slot) : nullptr;
            if (valid) {
                const size_t at = tree_row(p, sg, sg.row0 + r, D);
                float any[4] = {0.f, 0.f, 0.f, 0.f};  // NaN where a column is not finite
#pragma unroll
                for (int u = 0; u < D / 2; ++u) any[u & 3] = fmaf(o[u], 0.f, any[u & 3]);
                any[0] = (any[0] + any[1]) + (any[2] + any[3]);
                if (__builtin_expect((odd || any[0] != any[0]) && l == l, 0)) {
                    const TreeSpan a = {sg.seq, sg.head, (sg.row0 + r) / p.group, sg.t0 * BN, sg.t1 * BN, sg.s};
#pragma unroll
                    for (int c = 0; c < D / 2; c += 32) {
                        float tmp[32];  // its address is taken, o's is not
#pragma unroll
                        for (int u = 0; u < 32; ++u) tmp[u] = o[c + u];
                        tree_nonfinite<D, float>(p, a, half * (D / 2) + c, 32, any[0] != any[0], tmp);
#pragma unroll
                        for (int u = 0; u < 32; ++u) o[c + u] = tmp[u];
                    }
                }
                if (part) {
                    float4 *dst = reinterpret_cast<float4 *>(part) + (size_t)half * (D / 8) * p.rpg + r;
#pragma unroll
                    for (int u = 0; u < D / 8; ++u) dst[(size_t)u * p.rpg] = make_float4(o[4 * u], o[4 * u + 1], o[4 * u + 2], o[4 * u + 3]);
                    if (half == 0) {
                        part[(size_t)p.rpg * D + r] = m;
                        part[(size_t)p.rpg * (D + 1) + r] = l;
                    }
                } else {
                    float4 *dst = reinterpret_cast<float4 *>(static_cast<float *>(p.out) + at + half * (D / 2));
#pragma unroll
                    for (int u = 0; u < D / 8; ++u)
                        dst[u] = make_float4(o[4 * u] * inv, o[4 * u + 1] * inv, o[4 * u + 2] * inv, o[4 * u + 3] * inv);
                }
            }
            __syncwarp();
            ++segs;
        }
    } else {
        // --------------------------------------------------------- K and V split
        const uint32_t cw = warp - 2 - kRowWarps, tid = cw * 32 + lane;
        constexpr uint32_t kN = kSplitWarps * 32;
        uint32_t total = 0;  // tiles of this CTA
        {
            TreeWalk<false> w(range);
            TreeSeg g;
            while (w.next(p, g)) total += g.t1 - g.t0;
        }
        auto split_k = [&](uint32_t i) {
            wait_bar(&sh.k_full[i & 1u], (i >> 1) & 1u, abort_flag, p.wait_ns);
            __syncwarp();
            uint4 *k = reinterpret_cast<uint4 *>(smem + C::OFF_K + (i & 1u) * 2 * C::TILE);
#pragma unroll 4
            for (uint32_t x = tid; x < C::TILE / 16; x += kN) {
                constexpr uint32_t kBlock = BN * 8;  // 16-byte pieces of a block's hi (or lo) rows
                const uint32_t e = x + x / kBlock * kBlock;
                const uint4 y = k[e];
                uint4 h, l;
                tf32_split_any(__uint_as_float(y.x), h.x, l.x);
                tf32_split_any(__uint_as_float(y.y), h.y, l.y);
                tf32_split_any(__uint_as_float(y.z), h.z, l.z);
                tf32_split_any(__uint_as_float(y.w), h.w, l.w);
                k[e] = h;
                k[e + kBlock] = l;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.k_ready[i & 1u]);
        };
        if (total) split_k(0);
        while (walk.next(p, sg)) {
            const uint32_t P = sg.s.L - min(sg.s.T, sg.s.L);
            for (uint32_t j = sg.t0; j < sg.t1; ++j, ++it) {
                // V(it) transposed: thread = 4 positions of one column
                wait_bar(&sh.v_full, it & 1u, abort_flag, p.wait_ns);
                if (it > 0) wait_bar(&sh.o_full, (it & 1u) ^ 1u, abort_flag, p.wait_ns);  // the last tile's V has been read
                __syncwarp();
                const float *v = reinterpret_cast<const float *>(smem + C::OFF_V);
                const uint32_t kv0 = j * BN;
                const bool edge = kv0 + BN > P;
#pragma unroll 4
                for (uint32_t u = cw; u < BN / 4 * (D / 32); u += kSplitWarps) {
                    const uint32_t quad = u % (BN / 4), d = u / (BN / 4) * 32 + lane;
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = v[(quad * 4 + e) * D + d];
                    if (edge) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t pos = kv0 + quad * 4 + e;
                            if (pos >= sg.s.L) x[e] = 0.f;
                            else if (pos >= P && !(fabsf(x[e]) < INFINITY)) {
                                x[e] = 0.f;
                                *(volatile uint32_t *)&sh.odd[segs % 3] = segs + 1;
                            }
                        }
                    }
                    uint4 h, l;
                    tf32_split_any(x[0], h.x, l.x);
                    tf32_split_any(x[1], h.y, l.y);
                    tf32_split_any(x[2], h.z, l.z);
                    tf32_split_any(x[3], h.w, l.w);
                    const uint32_t to = (quad >> 3) * (D * 128) + d * 128 + (((quad & 7) ^ (d & 7)) << 4);
                    *reinterpret_cast<uint4 *>(smem + C::OFF_VHI + to) = h;
                    *reinterpret_cast<uint4 *>(smem + C::OFF_VLO + to) = l;
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&sh.v_empty);
                    mbar_arrive(&sh.v_ready);
                }
                if (it + 1 < total) split_k(it + 1);
            }
            ++segs;
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM_COLS) : "memory");
    }
}

// (d, n_kv, rows) view of a pool.
bool pool_map(CUtensorMap *map, const void *base, uint32_t d, uint32_t n_kv, uint64_t rows, uint32_t box_d, uint32_t box_rows,
              CUtensorMapSwizzle swizzle) {
    auto enc = get_encode();
    if (!enc) return false;
    cuuint64_t dims[3] = {d, n_kv, rows};
    cuuint64_t strides[2] = {(cuuint64_t)d * 4, (cuuint64_t)d * n_kv * 4};
    cuuint32_t box[3] = {box_d, 1, box_rows};
    cuuint32_t estr[3] = {1, 1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<void *>(base), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D>
cudaError_t launch_x(const TreeArgs &a, cudaStream_t st) {
    using C = XCfg<D>;
    static thread_local XParams xp;
    xp.t = a.p;
    const uint32_t page = 1u << a.p.page_shift;
    xp.box_rows = page < (uint32_t)BN ? page : (uint32_t)BN;
    xp.t.rpg = BM / a.p.group * a.p.group;
    xp.t.hpu = 1;
    xp.t.tile = BN;
    xp.t.heavy_rows = 0xffffffffu;
    xp.t.heavy = xp.t.light = 1;
    // 4 requests of 500 to 3000 positions: 37.4 us, 38.6 without a lead, 39.3 with 3; 40
    // of 50 to 1000: 52.8, 60.7, 55.8
    xp.t.lead = 1;
    if (!tree_line(xp.t)) return cudaErrorNotSupported;
    const uint64_t rows = (uint64_t)a.p.n_pages << a.p.page_shift;
    if (!pool_map(&xp.tk, a.p.k, D, a.p.n_kv, rows, 32, xp.box_rows, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !pool_map(&xp.tv, a.p.v, D, a.p.n_kv, rows, D, xp.box_rows, CU_TENSOR_MAP_SWIZZLE_NONE))
        return cudaErrorInvalidValue;
    auto kern = tree_umma32_kernel<D>;
    static SmemSet set;  // one for each instantiation
    cudaError_t e = set.allow(kern, C::SMEM);
    if (e != cudaSuccess) return e;
    e = launch_after(kern, dim3(a.num_sms), kThreads, C::SMEM, st, xp);
    if (e != cudaSuccess) return e;
    return launch_tree_merge(xp.t, D, a.num_sms, st);
}

}  // namespace

cudaError_t launch_tree_umma32(const TreeArgs &a, cudaStream_t st) { return a.D == 128 ? launch_x<128>(a, st) : launch_x<64>(a, st); }

}  // namespace bml
