// tree_umma.cu -- attention of drafted tokens over a paged cache on tcgen05
// tensor cores (sm_100a): 16-bit queries over pages of their type.
//
// The mathematics and the schedule are those of tree.cu / tree.cuh: a CTA
// (one per SM) works through its even share of the line of 128-position
// tiles, segment by segment.  A segment is a run of tiles of one unit (one
// request, kv head and group of up to 2 * RT query rows, RT = the most whole
// tokens' rows that fit 128).  Row r of a unit is (node r / group, q head
// r % group), so the q heads that share a kv head share its K and V tiles.
//
// Two chains, A and B, alternate on the tensor core, each with its own S
// (128 x 128) and O (128 x D) in tensor memory:
//   rows > RT:  A and B hold the unit's two row tiles and see every K/V tile;
//   rows <= RT: both hold the same rows, A sees even tiles and B odd ones,
//               and the epilogue joins them.
// While the softmax of one chain runs, the tensor core works for the other.
//   warp 0      producer: Q row tiles, then K and V tiles through one ring of
//               tile slots in the order the MMAs read them; a tile is one
//               cp.async.bulk.tensor per page and 128-byte column block.
//   warp 1      tensor memory, and every tcgen05.mma.
//   warps 2-5   softmax of A, warps 6-9 of B: thread = row = TMEM lane.
// All roles run over segment after segment with running barrier phases, so
// the copies of a segment's first tiles overlap the segment before.
//
// What a row does not see must not reach it: scores are replaced by -inf
// (bad pages, rows past the length, nodes outside the mask), V rows past the
// length are zeroed in shared memory before the first P.V that reads them,
// and so are V rows of drafted nodes with a value that is not finite (0 * NaN
// is not 0); the epilogue adds those nodes for the rows that see them.
#include <math.h>

#include "tree.cuh"
#include "umma.cuh"

namespace bml {

namespace {

constexpr int BM = 128;  // rows of a row tile (TMEM lanes)
constexpr int BN = kTreeTile;
constexpr int kThreads = 320;
constexpr float kRescaleThreshold = 8.0f;  // log2 units
constexpr int kBadRing = 16;               // tiles whose page flags are kept; more than the ring holds

template <int D>
struct UCfg {
    static constexpr int KB = D / 64;              // 128-byte column blocks of a row
    static constexpr int TILE = BM * D * 2;        // one Q, K or V tile
    static constexpr int SLOTS = D == 128 ? 5 : 11;  // K/V tile ring
    static constexpr int OFF_RING = 2 * TILE;
    static constexpr int OFF_BAR = OFF_RING + SLOTS * TILE;
    static constexpr int SMEM = OFF_BAR + 3072;  // + barriers and small arrays
    static constexpr uint32_t O_COL0 = 256;
    static constexpr uint32_t TMEM_COLS = 512;
};
static_assert(UCfg<128>::SMEM <= 227 * 1024 && UCfg<64>::SMEM <= 227 * 1024, "shared memory");
static_assert(UCfg<64>::SLOTS <= 2 * kBadRing && UCfg<128>::SLOTS <= 2 * kBadRing, "page flags");

struct UmmaParams {
    CUtensorMap tq, tk, tv;  // (d, heads, tokens) box (64, group, 128 / group); (d, n_kv, rows) box (64, 1, box_rows)
    TreeParams t;
    uint32_t rt;        // rows of a row tile: 128 / group * group
    uint32_t box_rows;  // min(page, 128)
};

// Small shared arrays behind the ring.
struct alignas(16) UmmaShared {
    uint64_t full[11], empty[11];
    uint64_t q_full, q_empty;
    uint64_t s_full[2];
    uint64_t p_full[4];   // [chain][half]
    uint64_t o_final[2];
    uint64_t drain;
    uint32_t tmem, abort;
    uint32_t bad[kBadRing];  // per tile: 16-position blocks on pages outside the pool
    uint32_t odd[8];         // drafted nodes whose V has a value that is not finite
    float2 ml[256];          // (m, l) of both chains' rows
    TreeShared sched;
};
static_assert(sizeof(UmmaShared) <= 3072, "small arrays");

// Slots of a segment's n tiles in ring order.  Two row tiles: K0 V0 K1 V1 ...;
// one row tile (chains alternate tiles): K0 K1 V0 K2 V1 ... V(n-1), the order
// in which the MMAs read them.
__device__ __forceinline__ uint32_t k_index(bool pair, uint32_t j) { return pair ? 2 * j : (j ? 2 * j - 1 : 0); }
__device__ __forceinline__ uint32_t v_index(bool pair, uint32_t j, uint32_t n) {
    return pair ? 2 * j + 1 : min(2 * j + 2, 2 * n - 1);
}

// Mask bits of nodes n0 .. n0 + 31 for node t of the request (n0 < 0: the
// committed positions before the nodes, seen by all).
__device__ __forceinline__ uint32_t see32(const TreeParams &p, const TreeSeq &s, uint32_t t, int32_t n0) {
    if (n0 >= (int32_t)s.T || s.L == 0) return 0u;
    if (n0 <= -32) return 0xffffffffu;
    const uint32_t first = n0 < 0 ? 0u : (uint32_t)n0;
    uint64_t w;  // bit i: node first + i
    if (p.mask) {
        const uint64_t *m = p.mask + (size_t)(s.first + t) * p.n_words;
        const uint32_t i = first >> 6, sh = first & 63;
        w = m[i] >> sh;
        if (sh > 32 && i + 1 < p.n_words) w |= m[i + 1] << (64 - sh);
    } else {
        const int32_t k = (int32_t)t - (int32_t)first;  // nodes up to t
        w = k < 0 ? 0ull : k >= 63 ? ~0ull : (2ull << k) - 1;
    }
    const uint32_t left = s.T - first;
    if (left < 32) w &= (1ull << left) - 1;
    if (n0 < 0) return (uint32_t)(w << -n0) | ((1u << -n0) - 1);
    return (uint32_t)w;
}

// 2^(scale q.k) of one row and one position, from global memory; for the rare
// nodes that the epilogue adds.
template <int D, bool kF16>
__device__ __noinline__ float rare_score(const uint16_t *q, const uint16_t *k) {
    float s = 0.f;
    for (int i = 0; i < D; ++i) {
        const float a = kF16 ? __half2float(reinterpret_cast<const __half *>(q)[i]) : __uint_as_float((uint32_t)q[i] << 16);
        const float b = kF16 ? __half2float(reinterpret_cast<const __half *>(k)[i]) : __uint_as_float((uint32_t)k[i] << 16);
        s = fmaf(a, b, s);
    }
    return s;
}

template <bool kF16>
__device__ __forceinline__ float one16(uint16_t x) {
    return kF16 ? __half2float(*reinterpret_cast<const __half *>(&x)) : __uint_as_float((uint32_t)x << 16);
}

template <int D, bool kF16>
__global__ void __launch_bounds__(kThreads, 1) tree_umma_kernel(const __grid_constant__ UmmaParams up) {
    using C = UCfg<D>;
    const TreeParams &p = up.t;
    // 1024-byte alignment for the 128B-swizzle atoms (there is no room for
    // slack; without static shared memory the array starts on such a boundary)
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t *ring = smem + C::OFF_RING;
    UmmaShared &sh = *reinterpret_cast<UmmaShared *>(smem + C::OFF_BAR);
    volatile uint32_t *abort_flag = &sh.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < C::SLOTS; ++i) {
            mbar_init(&sh.full[i], 1);
            mbar_init(&sh.empty[i], 1);
        }
        mbar_init(&sh.q_full, 1);
        mbar_init(&sh.q_empty, 1);
        for (int x = 0; x < 2; ++x) {
            mbar_init(&sh.s_full[x], 1);
            mbar_init(&sh.p_full[2 * x], 4);
            mbar_init(&sh.p_full[2 * x + 1], 4);
            mbar_init(&sh.o_final[x], 1);
        }
        mbar_init(&sh.drain, 1);
        sh.abort = 0u;
        fence_mbar_init();
    }
    if (threadIdx.x < 8) sh.odd[threadIdx.x] = 0u;
    if (warp == 0 && lane == 0) {
        prefetch_tmap(&up.tq);
        prefetch_tmap(&up.tk);
        prefetch_tmap(&up.tv);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)),
                     "r"(C::TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    const TreeRange range = tree_range(p, &sh.sched, blockIdx.x, gridDim.x);  // has the barriers for the set-up above
    tc_fence_after();
    const uint32_t tmem = *(volatile uint32_t *)&sh.tmem;
    TreeWalk walk(p, range);
    TreeSeg sg;

    if (warp == 0) {
        // ------------------------------------------------------------- producer
        uint32_t cnt = 0, tiles = 0, segs = 0;  // slots, tiles, segments so far
        const uint32_t per_tile = BN / up.box_rows, part = lane / C::KB, kb = lane % C::KB;
        const uint32_t ps_mask = (1u << p.page_shift) - 1;
        const bool mine = part < per_tile;
        auto wait_all = [&](uint64_t *bar, uint32_t parity) {
            bool ok = mbar_wait(bar, parity, abort_flag, nullptr);
            return __all_sync(0xffffffffu, ok);
        };
        bool live = true;
        while (live && walk.next(p, sg)) {
            const bool pair = sg.rows > up.rt;
            const uint32_t n = sg.t1 - sg.t0;
            if (segs > 0) live = wait_all(&sh.q_empty, (segs - 1) & 1u);
            if (!live) break;
            if (lane == 0) {
                const uint32_t tile_rows = up.rt;
                const uint32_t bytes = tile_rows * 128 * C::KB;
                mbar_arrive_expect_tx(&sh.q_full, bytes * (pair ? 2 : 1));
                const int tok = (int)(sg.s.first + sg.row0 / p.group);
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    if (x && !pair) break;
#pragma unroll
                    for (int b = 0; b < C::KB; ++b)
                        tma_load_3d(smem + x * C::TILE + b * BM * 128, &up.tq, b * 64, (int)(sg.head * p.group),
                                    tok + x * (int)(tile_rows / p.group), &sh.q_full);
                }
            }
            const int32_t *table = p.table + (size_t)sg.seq * p.max_pages;
            // row of the pools where this lane's box of tile j starts; -1: past the length, -2: not in the pool
            auto box_row = [&](uint32_t j) -> int {
                const uint32_t pos = (sg.t0 + j) * BN + part * up.box_rows;
                if (!mine || j >= n || pos >= sg.s.L) return -1;
                const uint32_t page = (uint32_t)table[pos >> p.page_shift];
                return page < p.n_pages ? (int)((page << p.page_shift) + (pos & ps_mask)) : -2;
            };
            auto issue = [&](bool is_k, int row) {
                const uint32_t slot = cnt % C::SLOTS;
                if (cnt >= (uint32_t)C::SLOTS && !wait_all(&sh.empty[slot], ((cnt / C::SLOTS) & 1u) ^ 1u)) return false;
                const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, row != -1));
                if (lane == 0) mbar_arrive_expect_tx(&sh.full[slot], boxes * up.box_rows * 128);
                __syncwarp();
                // a page outside the pool is read past the map's end: zeros
                if (row != -1)
                    tma_load_3d(ring + slot * C::TILE + kb * BN * 128 + part * up.box_rows * 128, is_k ? &up.tk : &up.tv,
                                (int)kb * 64, (int)sg.head, row == -2 ? (int)(p.n_pages << p.page_shift) : row, &sh.full[slot]);
                ++cnt;
                return true;
            };
            // rows of the tiles whose K, V come next; V trails K by one (two row tiles: none)
            int row_k = box_row(0), row_v = row_k;
            auto step_k = [&](uint32_t j) {
                const uint32_t bits = up.box_rows / 16;  // 16-position blocks of a box
                uint32_t flag = row_k == -2 ? ((1u << bits) - 1) << (part * bits) : 0u;
                flag = __reduce_or_sync(0xffffffffu, flag);
                if (lane == 0) *(volatile uint32_t *)&sh.bad[(tiles + j) % kBadRing] = flag;
                __syncwarp();
                return issue(true, row_k);
            };
            if (pair) {
                for (uint32_t j = 0; j < n && live; ++j) {
                    live = step_k(j);
                    row_v = row_k;
                    row_k = box_row(j + 1);
                    live = live && issue(false, row_v);
                }
            } else {
                live = step_k(0);
                for (uint32_t j = 0; j < n && live; ++j) {
                    row_v = row_k;
                    row_k = box_row(j + 1);
                    if (j + 1 < n) live = step_k(j + 1);
                    live = live && issue(false, row_v);
                }
            }
            tiles += n;
            ++segs;
        }
        // no copy may outlive the CTA (all have landed unless a wait gave up)
        for (uint32_t i = cnt > (uint32_t)C::SLOTS ? cnt - C::SLOTS : 0; i < cnt; ++i)
            mbar_drain(&sh.full[i % C::SLOTS], (i / C::SLOTS) & 1u, kWaitNs);
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------------------- MMA issuer
        constexpr uint32_t fmt = kF16 ? 0u : 1u;
        constexpr uint32_t idesc_qk = make_idesc(fmt, BM, BN, 0);
        constexpr uint32_t idesc_pv = make_idesc(fmt, BM, D, 1);
        const uint64_t dq = smem_desc(smem_u32(smem), 16, 1024);
        const uint64_t dk = smem_desc(smem_u32(ring), 16, 1024);
        const uint64_t dv = smem_desc(smem_u32(ring), BN * 128, 1024);
        uint32_t cnt = 0, segs = 0;
        uint32_t done[2] = {0, 0};  // tiles of each chain so far
        bool live = true;
        auto gate = [&](uint64_t *bar, uint32_t parity) {
            live = live && __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, nullptr));
            __syncwarp();
            tc_fence_after();
        };
        while (live && walk.next(p, sg)) {
            const bool pair = sg.rows > up.rt;
            const uint32_t n = sg.t1 - sg.t0;
            const uint32_t nt[2] = {pair ? n : (n + 1) / 2, pair ? n : n / 2};
            auto tile = [&](uint32_t x, uint32_t i) { return pair ? i : 2 * i + x; };
            auto qk = [&](uint32_t x, uint32_t i) {
                const uint32_t c = cnt + k_index(pair, tile(x, i)), slot = c % C::SLOTS;
                gate(&sh.full[slot], (c / C::SLOTS) & 1u);
                if (!live) return;
                const uint64_t a0 = dq + ((pair ? x * C::TILE : 0) >> 4), b0 = dk + ((slot * C::TILE) >> 4);
                const uint32_t d = tmem + x * 128;
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    const uint32_t off = ((kk >> 2) * (BM * 128) + (kk & 3) * 32) >> 4;
                    if (elect_one()) tc_mma_ss(d, a0 + off, b0 + off, idesc_qk, kk > 0);
                    __syncwarp();
                }
                if (elect_one()) {
                    tc_commit(&sh.s_full[x]);
                    if (!pair || x == 1) tc_commit(&sh.empty[slot]);
                }
                __syncwarp();
            };
            auto pv = [&](uint32_t x, uint32_t i) {
                const uint32_t c = cnt + v_index(pair, tile(x, i), n), slot = c % C::SLOTS;
                const uint64_t b0 = dv + ((slot * C::TILE) >> 4);
                const uint32_t d = tmem + C::O_COL0 + x * D, a = tmem + x * 128;
                const uint32_t par = (done[x] + i) & 1u;
                gate(&sh.full[slot], (c / C::SLOTS) & 1u);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    gate(&sh.p_full[2 * x + h], par);
                    if (!live) return;
#pragma unroll
                    for (int k4 = 0; k4 < BN / 32; ++k4) {
                        const int kk = h * (BN / 32) + k4;
                        if (elect_one())
                            tc_mma_ts(d, a + kk * 8, b0 + ((kk * 16 * 128) >> 4), idesc_pv, (kk > 0 || i > 0) ? 1u : 0u);
                        __syncwarp();
                    }
                }
                if (elect_one()) {
                    if (!pair || x == 1) tc_commit(&sh.empty[slot]);
                    if (i + 1 == nt[x]) tc_commit(&sh.o_final[x]);
                }
                __syncwarp();
            };
            gate(&sh.q_full, segs & 1u);
            uint32_t left = nt[0] + nt[1];  // S still to issue
            auto qk_last = [&](uint32_t x, uint32_t i) {
                qk(x, i);
                if (--left == 0) {  // the segment's Q has been read once this commit's MMAs are done
                    if (elect_one()) tc_commit(&sh.q_empty);
                    __syncwarp();
                }
            };
            if (live) qk_last(0, 0);
            if (live && nt[1]) qk_last(1, 0);
            for (uint32_t i = 0; i < nt[0] && live; ++i) {
#pragma unroll
                for (uint32_t x = 0; x < 2; ++x) {
                    if (i < nt[x] && live) {
                        pv(x, i);
                        if (i + 1 < nt[x] && live) qk_last(x, i + 1);
                    }
                }
            }
            cnt += 2 * n;
            done[0] += nt[0];
            done[1] += nt[1];
            ++segs;
        }
        if (elect_one()) tc_commit(&sh.drain);  // no MMA outlives the CTA
        __syncwarp();
        mbar_drain(&sh.drain, 0, kWaitNs);
        __syncwarp();
    } else {
        // ------------------------------------------------------------- softmax
        const uint32_t x = (uint32_t)(warp - 2) >> 2;
        const uint32_t q4 = warp & 3, r = q4 * 32 + lane;
        const uint32_t lane_addr = (q4 * 32) << 16;
        const uint32_t s_col = tmem + lane_addr + x * 128;
        const uint32_t o_base = tmem + lane_addr + C::O_COL0;
        const uint32_t o_col = o_base + x * D;
        const float c = p.scale_log2;
        uint32_t cnt = 0, tiles = 0, done = 0, finals = 0, finals_other = 0;
        while (walk.next(p, sg)) {
            const bool pair = sg.rows > up.rt;
            const uint32_t n = sg.t1 - sg.t0;
            const uint32_t nt = pair ? n : (x ? n / 2 : (n + 1) / 2);
            const uint32_t row = (pair ? x * up.rt : 0) + r;      // row of the group
            const bool valid = r < up.rt && row < sg.rows;
            const bool warp_live = __any_sync(0xffffffffu, valid);
            const uint32_t t = min((sg.row0 + row) / p.group, sg.s.T - 1);
            const uint32_t P = sg.s.L - min(sg.s.T, sg.s.L);
            float m_run = -INFINITY, l_run = 0.f;

            for (uint32_t i = 0; i < nt; ++i) {
                const uint32_t j = pair ? i : 2 * i + x;
                const uint32_t kv0 = (sg.t0 + j) * BN;
                mbar_wait(&sh.s_full[x], (done + i) & 1u, abort_flag, nullptr);
                __syncwarp();
                tc_fence_after();
                const uint32_t bad = *(volatile uint32_t *)&sh.bad[(tiles + j) % kBadRing];
                const bool edge = kv0 + BN > P;

                if (edge && (!pair || x == 0)) {
                    // V rows that must not be read as they are: this thread's row is kv0 + r
                    const uint32_t pos = kv0 + r, cv = cnt + v_index(pair, j, n), slot = cv % C::SLOTS;
                    if (__any_sync(0xffffffffu, pos >= P)) {
                        mbar_wait(&sh.full[slot], (cv / C::SLOTS) & 1u, abort_flag, nullptr);
                        uint8_t *vrow = ring + slot * C::TILE + r * 128;
                        bool zero = pos >= sg.s.L;
                        if (pos >= P && !zero) {
                            constexpr uint32_t em = kF16 ? 0x7c00u : 0x7f80u;
                            bool odd = false;
#pragma unroll
                            for (int u = 0; u < C::KB * 8; ++u) {
                                const uint4 w = lds128(vrow + (u >> 3) * BN * 128 + ((u + lane) & 7) * 16);
                                const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    odd |= (ws[e] & em) == em || ((ws[e] >> 16) & em) == em;
                            }
                            if (odd) {
                                atomicOr(&sh.odd[(pos - P) >> 5], 1u << ((pos - P) & 31));
                                zero = true;
                            }
                        }
                        if (zero) {
#pragma unroll
                            for (int u = 0; u < C::KB * 8; ++u)
                                *reinterpret_cast<uint4 *>(vrow + (u >> 3) * BN * 128 + ((u + lane) & 7) * 16) =
                                    make_uint4(0, 0, 0, 0);
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    }
                }
                if (!warp_live) {
                    // rows that nothing reads: P stays whatever S was
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(&sh.p_full[2 * x]);
                        mbar_arrive(&sh.p_full[2 * x + 1]);
                    }
                    continue;
                }
                float sv[BN];
#pragma unroll
                for (int cc = 0; cc < BN / 32; ++cc) tmem_ld32(s_col + cc * 32, sv + cc * 32);
                tmem_wait_ld();
                if (edge || bad) {
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        uint32_t see = edge ? see32(p, sg.s, t, (int32_t)(kv0 + 32 * w) - (int32_t)P) : 0xffffffffu;
                        if (bad >> (2 * w) & 1) see &= 0xffff0000u;
                        if (bad >> (2 * w + 1) & 1) see &= 0x0000ffffu;
#pragma unroll
                        for (int b = 0; b < 32; ++b)
                            if (!(see >> b & 1)) sv[w * 32 + b] = -INFINITY;
                    }
                }
                float mx8[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    float a = fmax3(sv[k], sv[k + 8], sv[k + 16]);
#pragma unroll
                    for (int u = 24; u < BN - 8; u += 16) a = fmax3(a, sv[k + u], sv[k + u + 8]);
                    mx8[k] = fmaxf(a, sv[k + BN - 8]);
                }
                const float mh = fmax3(fmax3(mx8[0], mx8[1], mx8[2]), fmax3(mx8[3], mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7]));
                // scale >= 0; with scale 0 a row that sees something has maximum 0
                const float m_tile = mh == -INFINITY ? -INFINITY : mh * c;
                float m_new = m_run;
                if (m_run == -INFINITY || m_tile > m_run + kRescaleThreshold) m_new = fmaxf(m_run, m_tile);
                const float m_use = (m_new == -INFINITY) ? 0.f : m_new;
                const float alpha = (m_run == -INFINITY) ? 0.f : fast_exp2(m_run - m_use);
                const bool rescale = (i > 0) && (m_new != m_run);
                m_run = m_new;

                const float2 c2 = make_float2(c, c), nm2 = make_float2(-m_use, -m_use);
                float2 sum4[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                for (int hv = 0; hv < 2; ++hv) {
#pragma unroll
                    for (int q2 = 0; q2 < 2; ++q2) {
                        const int qc = hv * 2 + q2;
                        uint32_t w[16];
#pragma unroll
                        for (int k = 0; k < 32; k += 2) {
                            float2 e = __ffma2_rn(make_float2(sv[qc * 32 + k], sv[qc * 32 + k + 1]), c2, nm2);
                            if (((k >> 1) & 7) == 7) {  // an eighth on the FMA pipe
                                e = exp2_poly_pair<true>(e);
                            } else {
                                e.x = fast_exp2(e.x);
                                e.y = fast_exp2(e.y);
                            }
                            sum4[(k >> 1) & 3] = __fadd2_rn(sum4[(k >> 1) & 3], e);
                            w[k >> 1] = pack2<kF16>(e.x, e.y);
                        }
                        tmem_st16(s_col + qc * 16, w);
                    }
                    if (hv == 0 && __any_sync(0xffffffffu, rescale)) {
                        const float a = rescale ? alpha : 1.f;
#pragma unroll
                        for (int cc = 0; cc < D / 32; ++cc) {
                            float o[32];
                            tmem_ld32(o_col + cc * 32, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int k = 0; k < 32; ++k) o[k] *= a;
                            tmem_st32(o_col + cc * 32, o);
                        }
                    }
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.p_full[2 * x + hv]);
                }
                const float2 sum2 = __fadd2_rn(__fadd2_rn(sum4[0], sum4[1]), __fadd2_rn(sum4[2], sum4[3]));
                l_run = l_run * alpha + (sum2.x + sum2.y);
            }
            if (m_run == -INFINITY && l_run == l_run) l_run = 0.f;  // saw nothing (a NaN stays)

            // --------------------------------------------------------- epilogue
            // One row tile: both chains' (m, l) meet in shared memory; chain x
            // writes columns x * D / 2 .. of the joined row.
            float wa, wb, m, l;  // row = wa * O_A + wb * O_B, un-normalised
            if (pair) {
                mbar_wait(&sh.o_final[x], finals & 1u, abort_flag, nullptr);
                wa = x == 0 && m_run > -INFINITY ? 1.f : 0.f;
                wb = x == 1 && m_run > -INFINITY ? 1.f : 0.f;
                m = m_run;
                l = l_run;
            } else {
                sh.ml[x * 128 + r] = make_float2(m_run, l_run);
                mbar_wait(&sh.o_final[0], (x == 0 ? finals : finals_other) & 1u, abort_flag, nullptr);
                if (n > 1) mbar_wait(&sh.o_final[1], (x == 1 ? finals : finals_other) & 1u, abort_flag, nullptr);
                __syncwarp();
                named_bar_sync(1, 256);
                const float2 a = sh.ml[r], b = sh.ml[128 + r];
                m = fmaxf(a.x, b.x);
                wa = a.x == -INFINITY ? 0.f : fast_exp2(a.x - m);
                wb = n < 2 || b.x == -INFINITY ? 0.f : fast_exp2(b.x - m);
                l = wa * a.y + wb * b.y;
            }
            __syncwarp();
            tc_fence_after();
            const bool gave_up = *abort_flag != 0u;
            const float inv = gave_up ? __int_as_float(0x7fffffff) : l == 0.f ? 0.f : 1.f / l;
            const uint32_t tt = (sg.row0 + row) / p.group;
            const size_t at = valid ? tree_row(p, sg, sg.row0 + row, D) : 0;
            float *part = sg.slot < 2 ? tree_part(p, D, blockIdx.x, sg.slot) : nullptr;
            const uint32_t first_cc = pair ? 0u : x * (D / 64), n_cc = pair ? D / 32 : D / 64;
            if (warp_live) {
#pragma unroll 1
                for (uint32_t k = 0; k < n_cc; ++k) {
                    const uint32_t cc = first_cc + k;
                    float o[32];
                    __syncwarp();
                    if (pair) {
                        tmem_ld32(o_col + cc * 32, o);
                        tmem_wait_ld();
                        const float w = wa + wb;
#pragma unroll
                        for (int u = 0; u < 32; ++u) o[u] = w == 0.f ? 0.f : o[u];
                    } else {
                        float o2[32];
                        tmem_ld32(o_base + cc * 32, o);
                        tmem_ld32(o_base + D + cc * 32, o2);
                        tmem_wait_ld();
#pragma unroll
                        for (int u = 0; u < 32; ++u) {
                            o[u] = wa == 0.f ? 0.f : o[u] * wa;
                            if (wb != 0.f) o[u] = fmaf(o2[u], wb, o[u]);
                        }
                    }
                    // nodes whose V was zeroed because a value is not finite
                    for (uint32_t node = 0; node < sg.s.T; ++node) {
                        if ((node & 31) == 0 && sh.odd[node >> 5] == 0u) {
                            node += 31;
                            continue;
                        }
                        const uint32_t pos = P + node;
                        if (!(sh.odd[node >> 5] >> (node & 31) & 1) || pos < sg.t0 * BN || pos >= sg.t1 * BN) continue;
                        if (!valid || !tree_sees(p, sg.s, tt, node)) continue;
                        const uint32_t page = (uint32_t)p.table[(size_t)sg.seq * p.max_pages + (pos >> p.page_shift)];
                        const size_t kvrow = ((((size_t)page << p.page_shift) + (pos & ((1u << p.page_shift) - 1))) * p.n_kv + sg.head) * D;
                        const float s = rare_score<D, kF16>(static_cast<const uint16_t *>(p.q) + at, static_cast<const uint16_t *>(p.k) + kvrow);
                        const float w = fast_exp2(s * c - m);
#pragma unroll 1
                        for (int u = 0; u < 32; ++u) {
                            const float v = one16<kF16>(static_cast<const uint16_t *>(p.v)[kvrow + cc * 32 + u]);
                            const float y = w * v;
#pragma unroll
                            for (int z = 0; z < 32; ++z)
                                if (z == u) o[z] += y;
                        }
                    }
                    if (valid && part) {
                        float4 *dst = reinterpret_cast<float4 *>(part + (size_t)row * D + cc * 32);
                        const float poison = gave_up ? inv : 1.f;
#pragma unroll
                        for (int u = 0; u < 8; ++u)
                            dst[u] = make_float4(o[4 * u] * poison, o[4 * u + 1] * poison, o[4 * u + 2] * poison, o[4 * u + 3] * poison);
                    } else if (valid) {
                        uint4 *dst = reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p.out) + at + cc * 32);
#pragma unroll
                        for (int u = 0; u < 4; ++u)
                            dst[u] = make_uint4(pack2<kF16>(o[8 * u] * inv, o[8 * u + 1] * inv),
                                                pack2<kF16>(o[8 * u + 2] * inv, o[8 * u + 3] * inv),
                                                pack2<kF16>(o[8 * u + 4] * inv, o[8 * u + 5] * inv),
                                                pack2<kF16>(o[8 * u + 6] * inv, o[8 * u + 7] * inv));
                    }
                }
                if (valid && part && (pair || x == 0)) {
                    part[(size_t)p.rpg * D + row] = m;
                    part[(size_t)p.rpg * (D + 1) + row] = l;
                }
            }
            tc_fence_before();
            __syncwarp();
            // The next segment's first P.V may overwrite O, its ml and odd words
            // be set, once both chains are here.
            const bool had_edge = sg.t1 * BN > P;
            if (!pair || had_edge) named_bar_sync(1, 256);
            if (had_edge) {
                if (threadIdx.x >= 64 && threadIdx.x < 72) sh.odd[threadIdx.x - 64] = 0u;
                __syncwarp();
                named_bar_sync(1, 256);
            }
            cnt += 2 * n;
            tiles += n;
            done += nt;
            if (nt) ++finals;
            if (pair || (x == 0 ? n / 2 : (n + 1) / 2)) ++finals_other;
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM_COLS) : "memory");
    }
}

// ----------------------------------------------------------------- host
// (d, heads, rows) view of a [rows][heads][d] 16-bit tensor.
bool tree_map(CUtensorMap *map, const void *base, bool f16, uint32_t d, uint32_t heads, uint64_t rows, uint32_t box_heads,
              uint32_t box_rows) {
    auto enc = get_encode();
    if (!enc) return false;
    cuuint64_t dims[3] = {d, heads, rows};
    cuuint64_t strides[2] = {(cuuint64_t)d * 2, (cuuint64_t)d * heads * 2};
    cuuint32_t box[3] = {64, box_heads, box_rows};
    cuuint32_t estr[3] = {1, 1, 1};
    return enc(map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(base), dims,
               strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool kF16>
cudaError_t launch_u(const UmmaParams &up, int num_sms, cudaStream_t st) {
    using C = UCfg<D>;
    auto kern = tree_umma_kernel<D, kF16>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return e;
    kern<<<num_sms, kThreads, C::SMEM, st>>>(up);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    return launch_tree_merge(up.t, D, num_sms, st);
}

}  // namespace

// A scale of 0 goes to the 32-bit form: here masked scores are scaled after they were set to -inf.
bool tree_umma_fits(const TreeArgs &a) { return a.kv_type != BML_F32 && a.p.q_type == a.kv_type && a.p.group <= (uint32_t)BM && a.p.scale_log2 > 0.f; }

cudaError_t launch_tree_umma(const TreeArgs &a, cudaStream_t st) {
    static thread_local UmmaParams up;
    up.t = a.p;
    const uint32_t group = a.p.group, page = 1u << a.p.page_shift;
    const bool f16 = a.kv_type == BML_F16;
    up.rt = BM / group * group;
    up.box_rows = page < (uint32_t)BN ? page : (uint32_t)BN;
    up.t.rpg = 2 * up.rt;
    up.t.min_tiles = 1;
    const uint64_t rows = (uint64_t)a.p.n_pages << a.p.page_shift;
    if (!tree_map(&up.tq, a.p.q, f16, a.D, a.p.n_heads, a.p.n_tokens, group, BM / group) ||
        !tree_map(&up.tk, a.p.k, f16, a.D, a.p.n_kv, rows, 1, up.box_rows) ||
        !tree_map(&up.tv, a.p.v, f16, a.D, a.p.n_kv, rows, 1, up.box_rows))
        return cudaErrorInvalidValue;
    if (a.D == 128) return f16 ? launch_u<128, true>(up, a.num_sms, st) : launch_u<128, false>(up, a.num_sms, st);
    return f16 ? launch_u<64, true>(up, a.num_sms, st) : launch_u<64, false>(up, a.num_sms, st);
}

}  // namespace bml
