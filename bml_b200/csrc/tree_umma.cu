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
//   warp 0      copies Q row tiles and K tiles, warp 10 V tiles: one ring of
//               tile slots in the order the MMAs read them; a tile is one
//               cp.async.bulk.tensor per page and 128-byte column block.
//   warp 1      tensor memory, and every tcgen05.mma.
//   warps 2-5   softmax of A, warps 6-9 of B: thread = row = TMEM lane.
// All roles run over segment after segment with running barrier phases, so
// the copies of a segment's first tiles overlap the segment before.  Warp 10
// also publishes the segments to the softmax warps, whose registers have no
// room for the walk.
//
// Measured on B200, 32 requests of 8000 positions, 32 / 8 heads, d = 128: 32
// nodes (128 rows) 186 us, 5.7 TB/s; 64 nodes (256 rows) 287 us, 940 TFLOP/s.
// 32 requests of 1024 to 8192, 16 to 64 nodes: tensor pipe busy 48% of the active
// cycles, the exponentials' unit 34%, issue 33%, each K and V byte read once: no
// unit is full, the chains wait for their softmax as in prefill.cu.
//
// What a row does not see must not reach it: scores are replaced by -inf
// (bad pages, rows past the length, nodes outside the mask), V rows past the
// length are zeroed in shared memory before the first P.V that reads them,
// and so are values of drafted nodes that are not finite (0 * NaN is not 0);
// tree_nonfinite adds those to the rows that see them.
#include <math.h>

#include <type_traits>

#include "tree.cuh"
#include "umma.cuh"

namespace bml {

namespace {

constexpr int BM = 128;  // rows of a row tile (TMEM lanes)
constexpr int BN = kTreeTile;
constexpr int kThreads = 352;  // K and Q producer, MMA issuer, 4 + 4 softmax warps, V producer
constexpr float kRescaleThreshold = 8.0f;  // log2 units
constexpr int kBadRing = 16;               // tiles whose page flags are kept; more than the ring holds

template <int D>
struct UCfg {
    static constexpr int KB = D / 64;              // 128-byte column blocks of a row
    static constexpr int TILE = BM * D * 2;        // one Q, K or V tile
    static constexpr int SLOTS = D == 128 ? 5 : 11;  // K/V tile ring
    static constexpr int OFF_RING = 2 * TILE;
    static constexpr int OFF_BAR = OFF_RING + SLOTS * TILE;
    static constexpr int SMEM = OFF_BAR + 3 * 1024;  // + barriers and small arrays
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

// One segment, as the softmax warps read it.
struct Board {
    uint32_t seq, first, T, L, head, row0, t0;
    uint32_t packed;  // tiles | slot << 28 | 1 << 31; 0: no more segments
};
// Entries of the ring of segments: the V producer is at most (slots / 2 + 2)
// segments ahead of the softmax.
constexpr uint32_t kBoard = 8;

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
    // [segment % 2]: the last segment (from 1 on) with a drafted node whose V has a
    // value that is not finite.  A chain is less than two segments ahead of the other.
    uint32_t odd[2];
    float2 ml[256];          // (m, l) of both chains' rows
    TreeShared sched;
    uint64_t seg_full[kBoard];
    Board board[kBoard];  // the segments, published by the V producer, which runs ahead
};
static_assert(sizeof(UmmaShared) <= 3 * 1024, "small arrays");

// Slots of a segment's n tiles in ring order.  Two row tiles: K0 V0 K1 V1 ...;
// one row tile (chains alternate tiles): K0 K1 V0 K2 V1 ... V(n-1), the order
// in which the MMAs read them.
__device__ __forceinline__ uint32_t k_index(bool pair, uint32_t j) { return pair ? 2 * j : (j ? 2 * j - 1 : 0); }
__device__ __forceinline__ uint32_t v_index(bool pair, uint32_t j, uint32_t n) {
    return pair ? 2 * j + 1 : min(2 * j + 2, 2 * n - 1);
}

// Which of a tile's 128 positions the row sees, as four words; node0: node of
// the tile's first position (negative: committed positions, seen by all).
// bad: 16-position blocks on pages outside the pool.  Out of line: few tiles
// need it, and the softmax's registers are dear.
__device__ __noinline__ uint4 see_tile(const TreeParams &p, const volatile Board *b, uint32_t row, int32_t node0, bool edge,
                                       uint32_t bad) {
    uint32_t see[4];
    const uint32_t T = b->T, L = b->L, t = min((b->row0 + row) / p.group, T - 1);
    const uint64_t *m = p.mask ? p.mask + (size_t)(b->first + t) * p.n_words : nullptr;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int32_t n0 = node0 + 32 * q;
        uint32_t s = 0xffffffffu;
        if (edge && (n0 >= (int32_t)T || L == 0)) s = 0u;
        else if (edge && n0 > -32) {
            const uint32_t first = n0 < 0 ? 0u : (uint32_t)n0;
            uint64_t w;  // bit i: node first + i
            if (m) {
                const uint32_t i = first >> 6, sh = first & 63;
                w = m[i] >> sh;
                if (sh > 32 && i + 1 < p.n_words) w |= m[i + 1] << (64 - sh);
            } else {
                const int32_t k = (int32_t)t - (int32_t)first;  // nodes up to t
                w = k < 0 ? 0ull : k >= 63 ? ~0ull : (2ull << k) - 1;
            }
            const uint32_t left = T - first;
            if (left < 32) w &= (1ull << left) - 1;
            s = n0 < 0 ? (uint32_t)(w << -n0) | ((1u << -n0) - 1) : (uint32_t)w;
        }
        if (bad >> (2 * q) & 1) s &= 0xffff0000u;
        if (bad >> (2 * q + 1) & 1) s &= 0x0000ffffu;
        see[q] = s;
    }
    return make_uint4(see[0], see[1], see[2], see[3]);
}

// One V row of a tile before its first P.V: zeros past the length, and in place
// of a drafted node's values that are not finite (then *odd = seg).  row: its
// first 128 bytes; the lanes start at different 16-byte pieces, against bank
// conflicts.
template <int KB, bool kF16>
__device__ __noinline__ void fix_v(uint8_t *row, bool node_row, bool past, volatile uint32_t *odd, uint32_t seg) {
    const uint32_t lane = threadIdx.x & 31;
    if (!node_row) return;
    constexpr uint32_t em = kF16 ? 0x7c00u : 0x7f80u;
    auto piece = [&](int u) { return reinterpret_cast<uint4 *>(row + (u >> 3) * BN * 128 + ((u + lane) & 7) * 16); };
    if (past) {
#pragma unroll 4
        for (int u = 0; u < KB * 8; ++u) *piece(u) = make_uint4(0, 0, 0, 0);
        return;
    }
    bool bad = false;
#pragma unroll 4
    for (int u = 0; u < KB * 8; ++u) {
        const uint4 w = lds128(reinterpret_cast<const uint8_t *>(piece(u)));
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) bad |= (ws[e] & em) == em || ((ws[e] >> 16) & em) == em;
    }
    if (!bad) return;
    *odd = seg;
#pragma unroll 1
    for (int u = 0; u < KB * 8; ++u) {
        const uint4 w = *piece(u);
        uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) ws[e] &= ((ws[e] & em) == em ? 0u : 0xffffu) | ((ws[e] >> 16 & em) == em ? 0u : 0xffff0000u);
        *piece(u) = make_uint4(ws[0], ws[1], ws[2], ws[3]);
    }
}

// tree_nonfinite for 32 columns of a row of node t.
template <int D, bool kF16>
__device__ __noinline__ void add_nonfinite(const TreeParams &p, const volatile Board *b, uint32_t t, uint32_t col, bool nan, float *o) {
    TreeSpan a = {b->seq, b->head, t, b->t0 * BN, (b->t0 + (b->packed & 0xfffffffu)) * BN, {}};
    a.s.first = b->first;
    a.s.T = b->T;
    a.s.L = b->L;
    tree_nonfinite<D, typename std::conditional<kF16, __half, __nv_bfloat16>::type>(p, a, col, 32, nan, o);
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
        for (uint32_t i = 0; i < kBoard; ++i) mbar_init(&sh.seg_full[i], 1);
        mbar_init(&sh.drain, 1);
        sh.abort = 0u;
        fence_mbar_init();
    }
    if (threadIdx.x < 2) sh.odd[threadIdx.x] = 0u;
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
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const TreeRange range = tree_range<true>(p, &sh.sched, blockIdx.x, gridDim.x);
    __syncthreads();  // the set-up above
    tc_fence_after();
    const uint32_t tmem = *(volatile uint32_t *)&sh.tmem;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the merge may take its place; it waits for this grid
    TreeWalk<true> walk(range);
    TreeSeg sg = {};

    if (warp == 0 || warp == 10) {
        // ------------------------------------------------------------- producers
        // Warp 0 copies Q and K, warp 10 V.  A lane issues one box: 128-byte
        // column block kb of part `part` of a tile.
        const bool is_k = warp == 0;
        const CUtensorMap *map = is_k ? &up.tk : &up.tv;
        const uint64_t policy = l2_policy_evict_first();
        uint32_t tiles = 0, segs = 0;  // tiles, segments so far
        uint32_t slot = 0, use = 0;    // ring position of the segment's next tile of either kind, and its use of the slot
        const uint32_t per_tile = BN / up.box_rows, part = lane / C::KB, kb = lane % C::KB;
        const uint32_t ps_mask = (1u << p.page_shift) - 1;
        const bool mine = part < per_tile;
        bool live = !(is_k && (p.diag & kTreeStall));
        auto wait_all = [&](uint64_t *bar, uint32_t parity) {
            live = live && __all_sync(0xffffffffu, wait_bar(bar, parity, abort_flag, p.wait_ns));
        };
        auto index = [&](bool pair, uint32_t j, uint32_t n) { return is_k ? k_index(pair, j) : v_index(pair, j, n); };
        auto advance = [&](uint32_t by) {  // at most 3
            slot += by;
            if (slot >= (uint32_t)C::SLOTS) {
                slot -= C::SLOTS;
                ++use;
            }
        };
        // The end is an entry of its own: every softmax warp sees the same
        // sequence, also when a wait gave up in the middle of a segment.
        uint32_t entries = 0;
        auto publish = [&](uint32_t more) {
            if (lane == 0) {
                Board &b = sh.board[entries % kBoard];
                if (more) b = Board{sg.seq, sg.s.first, sg.s.T, sg.s.L, sg.head, sg.row0, sg.t0, (sg.t1 - sg.t0) | sg.slot << 28 | 1u << 31};
                else b.packed = 0u;
                mbar_arrive(&sh.seg_full[entries % kBoard]);
            }
            ++entries;
            __syncwarp();
        };
        while (live && walk.next(p, sg)) {
            const bool pair = sg.rows > up.rt;
            const uint32_t n = sg.t1 - sg.t0;
            const int32_t *table = tree_table(p, sg.seq);
            // Table entries come 32 boxes at a time, one window ahead: lane l
            // holds the first row of box 32 w + l of the segment (-1: past the
            // length, -2: a page outside the pool).
            auto window = [&](uint32_t w) -> int {
                const uint32_t box = w * 32 + lane, pos = sg.t0 * BN + box * up.box_rows;
                if (box >= n * per_tile || pos >= sg.s.L) return -1;
                const uint32_t page = (uint32_t)table[pos >> p.page_shift];
                return page < p.n_pages ? (int)((page << p.page_shift) + (pos & ps_mask)) : -2;
            };
            int win = window(0), win_next = window(1);
            if (!is_k) publish(1u);
            if (is_k) {
                if (segs > 0) wait_all(&sh.q_empty, (segs - 1) & 1u);
                if (!live) break;
                // Q: a box per row tile and column block
                const uint32_t boxes = pair ? 2 * C::KB : C::KB;
                if (lane == 0) mbar_arrive_expect_tx(&sh.q_full, boxes * up.rt * 128);
                __syncwarp();
                if (lane < boxes) {
                    const uint32_t x = lane / C::KB, b = lane % C::KB;
                    tma_load_3d(smem + x * C::TILE + b * BM * 128, &up.tq, (int)b * 64, (int)(sg.head * p.group),
                                (int)(sg.s.first + (sg.row0 + x * up.rt) / p.group), &sh.q_full);
                }
                __syncwarp();
            }
            advance(index(pair, 0, n));
            for (uint32_t j = 0; j < n && live; ++j) {
                const uint32_t box = j * per_tile;
                if (j > 0 && (box & 31) == 0) {
                    win = win_next;
                    win_next = window(box / 32 + 1);
                }
                int row = __shfl_sync(0xffffffffu, win, (box + part) & 31);
                if (!mine) row = -1;
                if (is_k) {
                    const uint32_t bits = up.box_rows / 16;  // 16-position blocks of a box
                    uint32_t flag = 0;
                    if (__any_sync(0xffffffffu, row == -2))
                        flag = __reduce_or_sync(0xffffffffu, row == -2 ? ((1u << bits) - 1) << (part * bits) : 0u);
                    if (lane == 0) *(volatile uint32_t *)&sh.bad[(tiles + j) % kBadRing] = flag;
                }
                if (use > 0) wait_all(&sh.empty[slot], (use & 1u) ^ 1u);
                if (!live) break;
                const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, row != -1));
                if (lane == 0) mbar_arrive_expect_tx(&sh.full[slot], boxes * up.box_rows * 128);
                __syncwarp();
                // a page outside the pool is read past the map's end: zeros
                if (row != -1) {
                    uint8_t *dst = ring + slot * C::TILE + kb * BN * 128 + part * up.box_rows * 128;
                    const int at = row == -2 ? (int)(p.n_pages << p.page_shift) : row;
                    // with one row group K and V are read once: 7% faster out of HBM with the hint (32 x 8000, 32 nodes)
                    if (sg.s.groups == 1) tma_load_3d_hint(dst, map, (int)kb * 64, (int)sg.head, at, &sh.full[slot], policy);
                    else tma_load_3d(dst, map, (int)kb * 64, (int)sg.head, at, &sh.full[slot]);
                }
                __syncwarp();
                advance(j + 1 < n ? index(pair, j + 1, n) - index(pair, j, n) : 2 * n - index(pair, j, n));
            }
            tiles += n;
            ++segs;
        }
        if (!is_k) publish(0u);
        // No copy may outlive the CTA: all have landed unless a wait gave up,
        // and then none is issued any more, so those that have not will soon.
        if (!live) {
            const uint64_t t0 = globaltimer_ns();
            while (globaltimer_ns() - t0 < 1000000ull) {}
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------------------- MMA issuer
        constexpr uint32_t fmt = kF16 ? 0u : 1u;
        constexpr uint32_t idesc_qk = make_idesc(fmt, BM, BN, 0);
        constexpr uint32_t idesc_pv = make_idesc(fmt, BM, D, 1);
        const uint64_t dq = smem_desc(smem_u32(smem), 16, 1024);
        const uint64_t dk = smem_desc(smem_u32(ring), 16, 1024);
        const uint64_t dv = smem_desc(smem_u32(ring), BN * 128, 1024);
        // Slots are read in ring order; cur is the next one.
        struct Cursor {
            uint32_t slot, phase;
            __device__ __forceinline__ Cursor next() {
                const Cursor c = *this;
                if (++slot == (uint32_t)C::SLOTS) {
                    slot = 0;
                    phase ^= 1u;
                }
                return c;
            }
        };
        Cursor cur = {0, 0};
        uint32_t segs = 0, par = 0;  // par bit x: phase parity of chain x's P barriers
        bool live = true;
        // Before the last MMA of a block the barriers of the next block are
        // tested, so that a block whose operands are there follows without a gap.
        struct Gate {  // one or two barrier phases; b0 null: none
            uint64_t *b0;
            uint32_t p0;
            uint64_t *b1;
            uint32_t p1;
        };
        const Gate none = {nullptr, 0u, nullptr, 0u};
        auto full = [&](const Cursor &c) { return Gate{&sh.full[c.slot], c.phase, nullptr, 0u}; };
        auto p_half = [&](uint32_t x, uint32_t h) { return Gate{&sh.p_full[2 * x + h], par >> x & 1u, nullptr, 0u}; };
        auto gate_test = [&](const Gate &g) {
            bool ok = g.b0 == nullptr || mbar_test_wait(g.b0, g.p0);
            if (g.b1) ok = ok & mbar_test_wait(g.b1, g.p1);
            return ok;
        };
        auto gate_wait = [&](const Gate &g, bool ready) {
            if (!ready) {
                bool ok = true;
                if (g.b0) ok = wait_bar(g.b0, g.p0, abort_flag, p.wait_ns);
                if (g.b1) ok = wait_bar(g.b1, g.p1, abort_flag, p.wait_ns) && ok;
                live = live && __all_sync(0xffffffffu, ok);
            }
            __syncwarp();
            tc_fence_after();
        };
        // S of chain x from Q tile qt and the K tile in slot k
        auto qk = [&](uint32_t x, uint32_t qt, uint32_t k, bool release, bool last, const Gate &next) {
            const uint64_t a0 = dq + ((qt * C::TILE) >> 4), b0 = dk + ((k * C::TILE) >> 4);
            const uint32_t d = tmem + x * 128;
            bool ready = true;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
                if (kk == D / 16 - 1) ready = gate_test(next);
                const uint32_t off = ((kk >> 2) * (BM * 128) + (kk & 3) * 32) >> 4;
                if (elect_one()) tc_mma_ss(d, a0 + off, b0 + off, idesc_qk, kk > 0);
                __syncwarp();
            }
            if (elect_one()) {
                tc_commit(&sh.s_full[x]);
                if (release) tc_commit(&sh.empty[k]);
                if (last) tc_commit(&sh.q_empty);  // the segment's Q has been read
            }
            __syncwarp();
            return ready;
        };
        // O of chain x += P V over positions 64 h .. 64 h + 63 of the V tile in slot v
        auto pv = [&](uint32_t x, uint32_t v, int h, uint32_t acc, const Gate &next) {
            const uint64_t b0 = dv + ((v * C::TILE) >> 4);
            const uint32_t d = tmem + C::O_COL0 + x * D, a = tmem + x * 128;
            bool ready = true;
#pragma unroll
            for (int k4 = 0; k4 < BN / 32; ++k4) {
                const int kk = h * (BN / 32) + k4;
                if (k4 == BN / 32 - 1) ready = gate_test(next);
                if (elect_one()) tc_mma_ts(d, a + kk * 8, b0 + ((kk * 16 * 128) >> 4), idesc_pv, kk > 0 ? 1u : acc);
                __syncwarp();
            }
            return ready;
        };
        auto pv_done = [&](uint32_t x, uint32_t v, bool release, bool last) {
            if (elect_one()) {
                if (release) tc_commit(&sh.empty[v]);
                if (last) tc_commit(&sh.o_final[x]);
            }
            __syncwarp();
        };
        while (live && walk.next(p, sg)) {
            const uint32_t n = sg.t1 - sg.t0;
            Cursor k = cur.next();
            gate_wait(Gate{&sh.q_full, segs & 1u, &sh.full[k.slot], k.phase}, false);
            if (!live) break;
            if (sg.rows > up.rt) {
                // two row tiles: per K/V tile PV_A, S_A of the next, PV_B, S_B of the next
                qk(0, 0, k.slot, false, false, none);
                Cursor v = cur.next();
                Gate gv = {&sh.full[v.slot], v.phase, &sh.p_full[0], par & 1u};
                bool ready = qk(1, 1, k.slot, true, n == 1, gv);
                for (uint32_t i = 0; i < n; ++i) {
                    const bool more = i + 1 < n;
                    const uint32_t acc = i > 0;
                    gate_wait(gv, ready);
                    if (!live) break;
                    Gate g = p_half(0, 1);
                    gate_wait(g, pv(0, v.slot, 0, acc, g));
                    if (!live) break;
                    Gate gb = p_half(1, 0);
                    if (more) {
                        k = cur.next();
                        g = full(k);
                        ready = pv(0, v.slot, 1, acc, g);
                        gate_wait(g, ready);
                        if (!live) break;
                        ready = qk(0, 0, k.slot, false, false, gb);
                    } else {
                        ready = pv(0, v.slot, 1, acc, gb);
                        pv_done(0, v.slot, false, true);
                    }
                    gate_wait(gb, ready);
                    if (!live) break;
                    g = p_half(1, 1);
                    gate_wait(g, pv(1, v.slot, 0, acc, g));
                    if (!live) break;
                    pv(1, v.slot, 1, acc, none);
                    pv_done(1, v.slot, true, !more);
                    par ^= 3u;
                    if (more) {
                        v = cur.next();
                        gv = {&sh.full[v.slot], v.phase, &sh.p_full[0], par & 1u};
                        ready = qk(1, 1, k.slot, true, i + 2 == n, gv);
                    }
                }
            } else {
                // one row tile: chain j & 1 takes tile j; PV(j), then S(j + 2)
                bool ready;
                if (n > 1) {
                    const Cursor k1 = cur.next();
                    const Gate g = full(k1);
                    gate_wait(g, qk(0, 0, k.slot, true, false, g));
                    if (!live) break;
                    k = k1;
                }
                Cursor v = cur.next();
                Gate gv = {&sh.full[v.slot], v.phase, &sh.p_full[0], par & 1u};
                ready = qk(n > 1 ? 1 : 0, 0, k.slot, true, n < 3, gv);
                for (uint32_t j = 0; j < n; ++j) {
                    const uint32_t x = j & 1u, acc = j > 1;
                    gate_wait(gv, ready);
                    if (!live) break;
                    const Gate g = p_half(x, 1);
                    gate_wait(g, pv(x, v.slot, 0, acc, g));
                    if (!live) break;
                    const bool more = j + 2 < n;
                    const uint32_t vs = v.slot;
                    Gate gk = none;
                    if (more) {
                        k = cur.next();
                        gk = full(k);
                    }
                    ready = pv(x, vs, 1, acc, gk);
                    pv_done(x, vs, true, !more);
                    par ^= 1u << x;
                    if (more) {
                        gate_wait(gk, ready);
                        if (!live) break;
                    }
                    if (j + 1 < n) {
                        v = cur.next();
                        gv = {&sh.full[v.slot], v.phase, &sh.p_full[2 * (x ^ 1u)], par >> (x ^ 1u) & 1u};
                        ready = more ? qk(x, 0, k.slot, true, j + 3 == n, gv) : gate_test(gv);
                    }
                }
            }
            ++segs;
        }
        if (elect_one()) tc_commit(&sh.drain);  // no MMA outlives the CTA
        __syncwarp();
        mbar_drain(&sh.drain, 0, p.wait_ns);
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
        uint32_t cnt = 0, tiles = 0, done = 0, segs = 0;
        uint32_t finals = 0;  // bit x: phase parity of o_final[x]
        while (true) {
            // not cut short by the abort flag: the V producer's own waits are
            // bounded, and it always publishes an end; segments behind it (a wait
            // gave up) are tree_give_up's
            uint64_t *seg = &sh.seg_full[segs % kBoard];
            const uint32_t seg_phase = (segs / kBoard) & 1u;
            if (!mbar_test_wait(seg, seg_phase) && !mbar_drain(seg, seg_phase, 8 * p.wait_ns)) {
                *abort_flag = 1u;
                break;
            }
            __syncwarp();
            const volatile Board *b = &sh.board[segs % kBoard];
            const uint32_t packed = b->packed, n = packed & 0xfffffffu, slot_of = packed >> 28 & 7u;
            if (packed == 0u) break;
            const uint32_t rows = min(b->T * p.group - b->row0, p.rpg);
            const bool pair = rows > up.rt;
            const uint32_t nt = pair ? n : (x ? n / 2 : (n + 1) / 2);
            const uint32_t row = (pair ? x * up.rt : 0) + r;  // row of the group
            const bool valid = r < up.rt && row < rows;
            const bool warp_live = __any_sync(0xffffffffu, valid);
            const uint32_t P = b->L - min(b->T, b->L), kv_first = b->t0 * BN;
            float m_run = -INFINITY, l_run = 0.f;

            for (uint32_t i = 0; i < nt; ++i) {
                const uint32_t j = pair ? i : 2 * i + x;
                const uint32_t kv0 = kv_first + j * BN;
                wait_bar(&sh.s_full[x], (done + i) & 1u, abort_flag, p.wait_ns);
                __syncwarp();
                tc_fence_after();
                const uint32_t bad = *(volatile uint32_t *)&sh.bad[(tiles + j) % kBadRing];
                const bool edge = kv0 + BN > P;

                if (edge && (!pair || x == 0)) {
                    // V rows that must not be read as they are: this thread's row is kv0 + r
                    const uint32_t pos = kv0 + r, cv = cnt + v_index(pair, j, n), slot = cv % C::SLOTS;
                    if (__any_sync(0xffffffffu, pos >= P)) {
                        wait_bar(&sh.full[slot], (cv / C::SLOTS) & 1u, abort_flag, p.wait_ns);
                        fix_v<C::KB, kF16>(ring + slot * C::TILE + r * 128, pos >= P, pos >= b->L, &sh.odd[segs & 1u], segs + 1);
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
                uint4 see;  // before the scores are loaded: the call would spill them
                if (edge || bad) see = see_tile(p, b, row, (int32_t)(kv0 - P), edge, bad);
                float sv[BN];
#pragma unroll
                for (int cc = 0; cc < BN / 32; ++cc) tmem_ld32(s_col + cc * 32, sv + cc * 32);
                tmem_wait_ld();
                if (edge || bad) {
                    const uint32_t sees[4] = {see.x, see.y, see.z, see.w};
#pragma unroll
                    for (int w = 0; w < 4; ++w)
#pragma unroll
                        for (int k = 0; k < 32; ++k)
                            if (!(sees[w] >> k & 1)) sv[w * 32 + k] = -INFINITY;
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
                const float m_tile = mh * c;  // c > 0
                float m_new = m_run;
                if (m_run == -INFINITY || m_tile > m_run + kRescaleThreshold) m_new = fmaxf(m_run, m_tile);
                const float m_use = (m_new == -INFINITY) ? 0.f : m_new;
                const float alpha = (m_run == -INFINITY) ? 0.f : fast_exp2(m_run - m_use);
                const bool rescale = (i > 0) && (m_new != m_run);
                m_run = m_new;

                // P = 2^(s c - m) over S as packed 16-bit pairs, in two halves,
                // each released to the MMA warp as soon as it is written
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
                            if (!kF16 && ((k >> 1) & 7) == 7) w[k >> 1] = drop_tiny(w[k >> 1]);
                        }
                        tmem_st16(s_col + qc * 16, w);
                    }
                    if (hv == 0 && __any_sync(0xffffffffu, rescale)) {
                        const float a = rescale ? alpha : 1.f;
#pragma unroll 1
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
            // Row = wa * O_A + wb * O_B, un-normalised, with maximum m and sum l.
            // One row tile: both chains' (m, l) meet in shared memory, and chain x
            // writes columns x * D / 2 .. of the joined row.
            // has_a, has_b: the chain saw something (else its O may be anything).
            float wa, wb, m = m_run, l = l_run;
            bool has_a, has_b = false;
            if (pair) {
                wait_bar(&sh.o_final[x], (finals >> x) & 1u, abort_flag, p.wait_ns);
                has_a = m_run != -INFINITY;
                wa = 1.f;
                wb = 0.f;
            } else {
                sh.ml[x * 128 + r] = make_float2(m_run, l_run);
                wait_bar(&sh.o_final[0], finals & 1u, abort_flag, p.wait_ns);
                if (n > 1) wait_bar(&sh.o_final[1], finals >> 1 & 1u, abort_flag, p.wait_ns);
                __syncwarp();
                named_bar_sync(1, 256);
                const float2 ma = sh.ml[r], mb = sh.ml[128 + r];
                m = fmaxf(ma.x, mb.x);
                has_a = ma.x != -INFINITY;
                has_b = mb.x != -INFINITY;  // no tiles: -inf
                wa = has_a ? fast_exp2(ma.x - m) : 0.f;
                wb = has_b ? fast_exp2(mb.x - m) : 0.f;
                l = wa * ma.y + wb * mb.y;
            }
            __syncwarp();
            tc_fence_after();
            const bool gave_up = *abort_flag != 0u;
            if (gave_up) l = __int_as_float(0x7fffffff);
            const float inv = l == 0.f ? 0.f : 1.f / l;
            const uint32_t gr = b->row0 + row, t = gr / p.group;  // node; q head gr - t * group of the kv head
            const size_t at = valid ? ((size_t)(b->first + t) * p.n_heads + (size_t)b->head * p.group + (gr - t * p.group)) * D : 0;
            float *part = slot_of < 2 ? tree_part(p, D, blockIdx.x, slot_of) : nullptr;
            const bool odd = kv_first + n * BN > P && *(volatile uint32_t *)&sh.odd[segs & 1u] == segs + 1;
            if (warp_live) {
                const uint32_t first = pair ? 0u : x * (D / 2), n_cols = pair ? D : D / 2;
                const uint32_t src0 = pair ? o_col : o_base;
#pragma unroll 1
                for (uint32_t col = first; col < first + n_cols; col += 32) {
                    float o[32];
                    __syncwarp();
                    tmem_ld32(src0 + col, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int u = 0; u < 32; ++u) o[u] = has_a ? o[u] * wa : 0.f;
                    if (__any_sync(0xffffffffu, has_b)) {
                        float o2[32];
                        tmem_ld32(o_base + D + col, o2);
                        tmem_wait_ld();
                        if (has_b)
#pragma unroll
                            for (int u = 0; u < 32; ++u) o[u] = fmaf(o2[u], wb, o[u]);
                    }
                    if (valid) {
                        float any[4] = {0.f, 0.f, 0.f, 0.f};  // NaN where a column is not finite
#pragma unroll
                        for (int u = 0; u < 32; ++u) any[u & 3] = fmaf(o[u], 0.f, any[u & 3]);
                        any[0] = (any[0] + any[1]) + (any[2] + any[3]);
                        if (__builtin_expect((odd || any[0] != any[0]) && l == l, 0)) {
                            float tmp[32];  // its address is taken, o's is not
#pragma unroll
                            for (int u = 0; u < 32; ++u) tmp[u] = o[u];
                            add_nonfinite<D, kF16>(p, b, t, col, any[0] != any[0], tmp);
#pragma unroll
                            for (int u = 0; u < 32; ++u) o[u] = tmp[u];
                        }
                        if (part) {
                            float4 *dst = reinterpret_cast<float4 *>(part) + (size_t)(col / 4) * p.rpg + row;
#pragma unroll
                            for (int u = 0; u < 8; ++u) dst[u * p.rpg] = make_float4(o[4 * u], o[4 * u + 1], o[4 * u + 2], o[4 * u + 3]);
                        } else {
                            uint4 *dst = reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p.out) + at + col);
#pragma unroll
                            for (int u = 0; u < 4; ++u)
                                dst[u] = make_uint4(pack2<kF16>(o[8 * u] * inv, o[8 * u + 1] * inv),
                                                    pack2<kF16>(o[8 * u + 2] * inv, o[8 * u + 3] * inv),
                                                    pack2<kF16>(o[8 * u + 4] * inv, o[8 * u + 5] * inv),
                                                    pack2<kF16>(o[8 * u + 6] * inv, o[8 * u + 7] * inv));
                        }
                    }
                }
                if (valid && part && (pair || x == 0)) {
                    part[(size_t)p.rpg * D + row] = m;
                    part[(size_t)p.rpg * (D + 1) + row] = l;
                }
            }
            tc_fence_before();
            __syncwarp();
            // The next segment's first P.V may overwrite O, and its ml be set, once both
            // chains are here.
            if (!pair) named_bar_sync(1, 256);
            cnt += 2 * n;
            tiles += n;
            done += nt;
            finals ^= pair || n > 1 ? 3u : 1u;  // chains that had tiles
            ++segs;
        }
    }

    tc_fence_before();
    __syncthreads();
    if (*abort_flag) tree_give_up<true>(p, &sh.sched, D);
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
    static SmemSet set;  // one for each instantiation
    cudaError_t e = set.allow(kern, C::SMEM);
    if (e != cudaSuccess) return e;
    e = launch_after(kern, dim3(num_sms), kThreads, C::SMEM, st, up);
    if (e != cudaSuccess) return e;
    return launch_tree_merge(up.t, D, num_sms, st);
}

}  // namespace

bool tree_umma_fits(const TreeArgs &a) { return a.p.group <= (uint32_t)BM; }

cudaError_t launch_tree_umma(const TreeArgs &a, cudaStream_t st) {
    static thread_local UmmaParams up;
    up.t = a.p;
    const uint32_t group = a.p.group, page = 1u << a.p.page_shift;
    const bool f16 = a.kv_type == BML_F16;
    up.rt = BM / group * group;
    up.box_rows = page < (uint32_t)BN ? page : (uint32_t)BN;
    up.t.rpg = 2 * up.rt;
    up.t.hpu = 1;
    up.t.tile = kTreeTile;
    // A tile of two row tiles against one of one: measured on B200, d = 128, 32
    // requests of 8000 positions in L2: 2.4 us with 256 rows, 1.4 with 128.
    up.t.heavy_rows = up.rt;
    up.t.heavy = 5;
    up.t.light = 3;
    // 64 requests of 200 to 4000 positions, 4 to 16 nodes: 101 us, 130 without a lead,
    // 104 with 10, 103 with 40; 32 of 1024 to 8192, 16 to 64 nodes: 159, 172, 162, 156
    up.t.lead = 20;
    if (!tree_line(up.t)) return cudaErrorNotSupported;
    const uint64_t rows = (uint64_t)a.p.n_pages << a.p.page_shift;
    if (!tree_map(&up.tq, a.p.q, f16, a.D, a.p.n_heads, a.p.n_tokens, group, BM / group) ||
        !tree_map(&up.tk, a.p.k, f16, a.D, a.p.n_kv, rows, 1, up.box_rows) ||
        !tree_map(&up.tv, a.p.v, f16, a.D, a.p.n_kv, rows, 1, up.box_rows))
        return cudaErrorInvalidValue;
    if (a.D == 128) return f16 ? launch_u<128, true>(up, a.num_sms, st) : launch_u<128, false>(up, a.num_sms, st);
    return f16 ? launch_u<64, true>(up, a.num_sms, st) : launch_u<64, false>(up, a.num_sms, st);
}

}  // namespace bml
