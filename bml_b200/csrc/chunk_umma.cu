// chunk_umma.cu -- attention of chunks of new tokens over a paged cache on tcgen05
// tensor cores (sm_100a): 16-bit queries over pages of their type.
//
//   out[t] = sum_p softmax_p(scale q_t . k_p) v_p,  p = 0 .. P + t,  t = 0 .. T - 1
//
// A unit is one (request, kv head, row group): the rows (token t, q head g of the
// kv head) of tpg consecutive tokens, r = (t - t0) * group + g, in two row tiles of
// up to 128 rows.  A unit's tiles of 128 positions end at its last token's, so the
// masked half of a prompt costs nothing, and the q heads of a kv head share K and V.
//
// Schedule.  All units lie on one line, request by request, heads by heads, row
// group by row group, each with `lead` places for what its start and end cost and
// then its tiles.  The line is cut evenly over the CTAs (one an SM), so lengths and
// chunk sizes stay on the device and no CTA works longer than another by more than
// a tile.  A tile's place count is 128 times its weight, and a unit has weight *
// (positions + 127) of them -- a linear function of the row group, whose sums over
// groups have a closed form; the places behind the last tile are idle.  A unit that
// a cut divides leaves partial results that chunk_merge_kernel joins in tile order.
//
// Two chains, A and B, alternate on the tensor core, each with its own S (128 x
// 128) and O (128 x D) in tensor memory, as in prefill.cu:
//   rows > RT:  A and B hold the unit's two row tiles and see every K/V tile;
//   rows <= RT: both hold the same rows, A sees even tiles and B odd ones.
// Warps:
//   0      copies Q row tiles and K tiles, 2 V tiles (a cp.async.bulk.tensor per
//          page and 128-byte column block) through a ring each; 2 also walks the
//          schedule and publishes the CTA's segments to all others;
//   1, 3   tcgen05.mma of chain A and of chain B (1: tensor memory too);
//   4-11   softmax of A, 12-19 of B: two threads a row (TMEM lane), 64 scores each.
// One warp a chain issues its MMAs: a tcgen05.commit, or the wait for the next
// block's operands, holds the issuing warp up for longer than the tensor core has
// MMAs of N = 128 queued.  Measured on B200, 8 MMAs of 64 cycles and a commit in
// turn, with 16 other warps busy: 94 cycles an MMA from one warp, 65 from two.
// They take turns, P.V of a tile and S of the next, so that one chain's softmax runs
// while the tensor core works for the other.
//
// A chain's time a tile is its softmax and then its MMAs, so the softmax is kept short:
//   - two threads a row; with one (prefill.cu, tree_umma.cu) a scheduler's one warp of
//     the chain waits for its own exponentials and loads;
//   - it does not wait for a tile's maximum: it takes the exponentials of its first 32
//     scores against the maximum so far while the maximum is found beside them, and
//     only where that grew by more than 2^8 in either half (the result is exact for any
//     fixed reference) takes them anew, from tensor memory, and rescales O.
//
// Weights enter P.V rounded to the pages' 16-bit type, the only one that an MMA takes
// beside such a V: half a step of each, at most eps / 2 of the sum of p |v|.  Their sum
// stays f32 and takes them unrounded.
//
// Measured on B200, d = 128, group 4: 2048 tokens behind 30,720 positions 870 us alone
// and 990 to 1010 in a loop, at the power cap (1.22 to 1.05 PFLOP/s); 4 requests of 512
// behind 4000 155 us (920 TFLOP/s; tensor pipe 50% of active cycles, exponentials 51%: a
// chain's softmax and MMAs wait for each other); d = 64, 300 tokens behind 700 21 us, most
// of it start and end.
#include <math.h>

#include <type_traits>

#include "tree.cuh"
#include "umma.cuh"

namespace bml {

namespace {

constexpr int BM = 128;  // rows of a row tile (TMEM lanes)
constexpr int BN = kTreeTile;
constexpr int kThreads = 640;
constexpr uint32_t kSoftmaxWarps = 16;
constexpr float kRescaleThreshold = 8.0f;  // log2 units
constexpr int kBadRing = 16;               // tiles whose page flags are kept; more than the K ring holds
constexpr uint32_t kBoard = 4;             // segments that the schedule may be ahead

template <int D>
struct CCfg {
    static constexpr int KB = D / 64;              // 128-byte column blocks of a row
    static constexpr int TILE = BM * D * 2;        // one Q, K or V tile
    // Tiles of either ring.  Even, so that with one row tile, whose tiles the chains
    // take in turns, a slot's tiles are all one chain's: a chain that waits for a slot
    // has then seen the slot's phase before (a parity tells two phases apart only).
    static constexpr int STAGES = D == 128 ? 2 : 4;
    static constexpr int OFF_K = 2 * TILE, OFF_V = OFF_K + STAGES * TILE;
    static constexpr int OFF_BAR = OFF_V + STAGES * TILE;
    static constexpr int SMEM = OFF_BAR + 3 * 1024;  // + barriers and small arrays
    static constexpr uint32_t O_COL0 = 256;
    static constexpr uint32_t TMEM_COLS = 512;
};
static_assert(CCfg<128>::SMEM <= 227 * 1024 && CCfg<64>::SMEM <= 227 * 1024, "shared memory");
static_assert(CCfg<64>::STAGES % 2 == 0 && CCfg<128>::STAGES % 2 == 0, "rings");
constexpr int kMaxStages = 4;

struct ChunkParams {
    CUtensorMap tq, tk, tv;  // (d, heads, tokens) box (64, group, 128 / group); (d, n_kv, rows) box (64, 1, box_rows)
    TreeParams t;
    uint32_t rt;        // rows of a row tile: 128 / group * group
    uint32_t tpg;       // tokens of a row group: 2 * (128 / group)
    uint32_t box_rows;  // min(page, 128)
    uint32_t most_phases;
    struct ChunkCut *cuts;  // [most_phases * CTAs]
};
// What the merge reads of the unit that is divided behind piece i of the line and
// begins in it (rows 0: there is none): rows row0 .. of a request's kv head, with
// partial results of the pieces i .. last.
struct ChunkCut {
    uint32_t first, head, row0, rows, last, pad[3];
};

// ---------------------------------------------------------------------------
// Schedule
// ---------------------------------------------------------------------------
// A tile of two row tiles against one of one, and a unit's start and end in places
// (of a 128th of a weight).
constexpr uint64_t kHeavy = 2, kLight = 1, kLead = 8 * 128;

struct ChunkSeq {
    uint32_t first, T;   // token rows
    int32_t P;           // committed positions; far below 0: refused, its rows see nothing
    uint32_t groups;
    bool ok;
    uint64_t step, slope;  // F(k) = k step + slope k (k + 1) / 2: places of the first k row groups (not of the last)
    uint64_t places;       // of a head
    // positions that the row group's last token sees (1: refused)
    __device__ __forceinline__ uint32_t end(uint32_t rg, uint32_t tpg) const {
        return ok ? (uint32_t)P + min(T, (rg + 1) * tpg) : 1u;
    }
    __device__ __forceinline__ uint64_t before(uint32_t k) const { return k * step + slope * ((uint64_t)k * (k + 1) / 2); }
};

__device__ __forceinline__ uint64_t chunk_weight(const ChunkParams &p, uint32_t rows) { return rows > p.rt ? kHeavy : kLight; }

__device__ __forceinline__ ChunkSeq chunk_seq(const ChunkParams &p, uint32_t i, uint32_t lead) {
    const TreeRaw raw = tree_raw<false>(p.t, i);
    ChunkSeq s;
    const bool rows_ok = raw.a >= 0 && raw.b > raw.a && (uint32_t)raw.b <= p.t.n_tokens;
    s.first = rows_ok ? (uint32_t)raw.a : 0u;
    s.T = rows_ok ? (uint32_t)(raw.b - raw.a) : 0u;
    s.ok = raw.L >= (int32_t)s.T && (uint64_t)raw.L <= ((uint64_t)p.t.max_pages << p.t.page_shift);
    s.P = s.ok ? raw.L - (int32_t)s.T : -(1 << 30);
    s.groups = (s.T + p.tpg - 1) / p.tpg;
    s.step = kHeavy * ((s.ok ? (uint32_t)s.P : 1u) + 127u) + lead;
    s.slope = s.ok ? kHeavy * p.tpg : 0u;
    s.places = 0;
    if (s.groups) {
        const uint32_t rows = (s.T - (s.groups - 1) * p.tpg) * p.t.group;
        s.places = s.before(s.groups - 1) + chunk_weight(p, rows) * (s.end(s.groups - 1, p.tpg) + 127u) + lead;
    }
    return s;
}

// Out of line, and in 32 bits where they are enough: a launch meets this code cold.
__device__ __noinline__ uint64_t chunk_div(uint64_t a, uint64_t b) {
    if (((a | b) >> 32) == 0) return (uint32_t)a / (uint32_t)b;
    return a / b;
}

constexpr uint32_t kMostPhases = 4;
// K and V bytes of the requests with several row groups that a phase is meant to
// have.  Measured on B200 (L2 of 126 MB): 134 MB in one phase 958 us, in two 892, in
// three 870 to 895; 74 MB in one 170, in two 185.
constexpr uint64_t kPhaseBytes = 80ull << 20;

// The line of `total` places, cut into `active` pieces (a CTA's of each phase, at
// least a heavy tile each): the first `more` take one place more than the others.  A
// tile belongs to the piece in which it begins.
struct ChunkLine {
    uint64_t total, each, more;
    uint32_t phases, active, lead;
    __device__ __forceinline__ void cut(uint32_t pieces) {
        active = total >= pieces * kHeavy * BN ? pieces : max((uint32_t)total / (uint32_t)(kHeavy * BN), total ? 1u : 0u);
        each = active ? chunk_div(total, active) : 0u;
        more = total - each * active;
    }
    __device__ __forceinline__ uint64_t at(uint32_t piece) const { return each * piece + min((uint64_t)piece, more); }
    __device__ __forceinline__ uint32_t owner(uint64_t w) const {
        const uint64_t wide = more * (each + 1);
        return (uint32_t)(w < wide ? chunk_div(w, each + 1) : more + chunk_div(w - wide, each));
    }
};

// What the schedule's warp finds at the start: the line, and for each of the CTA's
// pieces the request that holds its first place, and that request's first place.
struct ChunkStarts {
    ChunkLine line;
    uint64_t base[kMostPhases];
    uint32_t seq[kMostPhases];
};

// By one warp: a lane takes a run of requests.
__device__ __forceinline__ void chunk_find(const ChunkParams &p, uint32_t D, ChunkStarts *out) {
    const uint32_t lane = threadIdx.x & 31, n = p.t.n_seqs;
    const uint32_t per = (n + 31) / 32, i0 = min(lane * per, n), i1 = min(i0 + per, n);
    uint64_t mine = 0, units = 0, again = 0;  // again: positions that are read more than once
#pragma unroll 4
    for (uint32_t i = i0; i < i1; ++i) {
        const ChunkSeq s = chunk_seq(p, i, 0);
        mine += s.places * p.t.n_kv;
        units += (uint64_t)s.groups * p.t.n_kv;
        if (s.groups > 1 && s.ok) again += (uint32_t)s.P + s.T;
    }
    uint64_t inc = mine, inc_units = units;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t a = __shfl_up_sync(0xffffffffu, inc, o), b = __shfl_up_sync(0xffffffffu, inc_units, o);
        const uint64_t c = __shfl_xor_sync(0xffffffffu, again, o);
        if (lane >= (uint32_t)o) {
            inc += a;
            inc_units += b;
        }
        again += c;
    }
    ChunkLine line;
    line.total = __shfl_sync(0xffffffffu, inc, 31);
    line.phases = 1;
    again *= 4ull * D * p.t.n_kv;
    while (line.phases < p.most_phases && again > kPhaseBytes * line.phases) ++line.phases;
    // no more than a piece's share, or whole pieces would fall into leads (3 requests of 90
    // tokens behind 300: 25.6 us, 27.5 without this, 26.5 with half the share)
    line.lead = (uint32_t)min((uint64_t)kLead, chunk_div(line.total, (uint64_t)line.phases * gridDim.x));
    line.total += line.lead * __shfl_sync(0xffffffffu, inc_units, 31);
    inc += line.lead * inc_units;
    mine += line.lead * units;
    line.cut(line.phases * gridDim.x);
    if (lane < kMostPhases) out->seq[lane] = n;
    if (lane == 0) out->line = line;
    __syncwarp();
    for (uint32_t k = 0; k < line.phases; ++k) {
        const uint32_t piece = k * gridDim.x + blockIdx.x;
        const uint64_t w0 = line.at(piece);
        uint64_t base = inc - mine;
        if (piece < line.active && w0 >= base && w0 < inc) {
            uint32_t i = i0;
            while (i + 1 < i1) {
                const uint64_t x = chunk_seq(p, i, line.lead).places * p.t.n_kv;
                if (w0 < base + x) break;
                base += x;
                ++i;
            }
            out->seq[k] = i;
            out->base[k] = base;
        }
    }
    __syncwarp();
}

// Consecutive tiles of one unit.
struct ChunkSeg {
    uint32_t seq, head, rg;
    uint32_t t0, t1;     // tiles [t0, t1) of the unit's `tiles`
    uint32_t tiles;
    uint64_t u0, w;      // the place of the unit's first tile, a tile's weight
    uint32_t row0, rows;
    uint32_t slot;       // partial slot of the piece: 0 the unit began before, 1 it ends after, 2 whole
    ChunkSeq s;
};

// The segments of a CTA's pieces in order.
struct ChunkWalk {
    uint64_t pos, end, base;
    uint32_t seq, phase;
    ChunkLine line;
    ChunkSeq s;
    __device__ __forceinline__ uint32_t piece() const { return phase * gridDim.x + blockIdx.x; }
    __device__ __forceinline__ void begin(const ChunkParams &p, const ChunkStarts *starts) {
        seq = starts->seq[phase];
        base = starts->base[phase];
        pos = end = 0;
        if (seq < p.t.n_seqs) {
            pos = line.at(piece());
            end = line.at(piece() + 1);
            s = chunk_seq(p, seq, line.lead);
        }
    }
    // the next segment of the piece
    __device__ __forceinline__ bool next(const ChunkParams &p, ChunkSeg &g) {
        while (pos < end) {
            while (pos - base >= s.places * p.t.n_kv) {
                base += s.places * p.t.n_kv;
                if (++seq >= p.t.n_seqs) {  // only with a node_start that does not ascend
                    pos = end;
                    return false;
                }
                s = chunk_seq(p, seq, line.lead);
            }
            const uint64_t off = pos - base;
            const uint32_t head = (uint32_t)chunk_div(off, s.places);
            const uint64_t in_head = off - head * s.places;
            uint32_t lo = 0, hi = s.groups;  // the last row group that begins at in_head or before
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) >> 1;
                if (s.before(mid) <= in_head) lo = mid;
                else hi = mid;
            }
            g.rg = lo;
            g.row0 = lo * p.tpg * p.t.group;
            g.rows = min(p.tpg, s.T - lo * p.tpg) * p.t.group;
            const uint32_t last = s.end(lo, p.tpg);
            g.tiles = (last + BN - 1) / BN;
            g.w = chunk_weight(p, g.rows);
            const uint64_t in = in_head - s.before(lo), len = line.lead + g.w * (last + 127u);
            const uint64_t out = min(in + (end - pos), len);
            // tiles that begin in [0, x): a tile's places, 128 w, divided in two steps
            auto first_at = [&](uint64_t x) {
                if (x <= line.lead) return 0u;
                const uint32_t y = (uint32_t)((x - line.lead + BN - 1) / BN);  // below 2^31 * 5 / 128
                return min(g.w == kHeavy ? (y + (uint32_t)kHeavy - 1) / (uint32_t)kHeavy : (y + (uint32_t)kLight - 1) / (uint32_t)kLight, g.tiles);
            };
            g.t0 = first_at(in);
            g.t1 = first_at(out);
            g.u0 = pos - in + line.lead;
            pos += out - in;
            if (g.t0 >= g.t1) continue;  // no tile begins here
            g.seq = seq;
            g.s = s;
            g.head = head;
            g.slot = g.t0 > 0 ? 0u : (g.t1 < g.tiles ? 1u : 2u);
            return true;
        }
        return false;
    }
};

__device__ __forceinline__ size_t chunk_slot(const ChunkParams &p, uint32_t D) { return ((size_t)2 * p.rt * (D + 2) + 3) & ~(size_t)3; }
// Partial slot i: 2 * piece + (0: the unit began before the piece, 1: it ends after).
__device__ __forceinline__ float *chunk_part(const ChunkParams &p, uint32_t D, uint32_t i) { return p.t.part + i * chunk_slot(p, D); }
// The record of a segment that is its unit's first and not its last.
__device__ __forceinline__ ChunkCut chunk_cut(const ChunkParams &p, const ChunkLine &line, const ChunkSeg &g) {
    return {g.s.first, g.head, g.row0, g.rows, line.owner(g.u0 + (uint64_t)(g.tiles - 1) * g.w * BN), {}};
}
// Element index of row r (token * group + g) of a request's kv head in q and out.
__device__ __forceinline__ size_t chunk_row(const ChunkParams &p, uint32_t first, uint32_t head, uint32_t r, uint32_t D) {
    const uint32_t t = r / p.t.group;
    return ((size_t)(first + t) * p.t.n_heads + (size_t)head * p.t.group + (r - t * p.t.group)) * D;
}

// ---------------------------------------------------------------------------
// Kernel
// ---------------------------------------------------------------------------
// One segment, as the warps read it.
struct Board {
    uint32_t seq, first, T;
    int32_t P;
    uint32_t head, row0, t0;
    uint32_t n;     // tiles; 0: no more segments
    uint32_t part;  // partial slot, kWhole: none
};
constexpr uint32_t kWhole = 0xffffffffu;

// Small shared arrays behind the ring.
struct alignas(16) ChunkShared {
    uint64_t k_full[kMaxStages], k_empty[kMaxStages], v_full[kMaxStages], v_empty[kMaxStages];
    uint64_t q_full, q_empty;
    uint64_t s_full[2];
    uint64_t p_full[4];  // [chain][step]: P of 32 positions of either half
    uint64_t o_final[2];
    uint64_t drain[2], turn[2];  // [chain]
    uint64_t seg_full[kBoard], seg_empty[kBoard];
    uint32_t tmem, abort;
    uint32_t bad[kBadRing];  // per tile: 16-position blocks on pages outside the pool
    // [chain][segment % 8]: the last segment (from 1 on) in which the chain met a masked
    // place whose V has a value that is not finite.  A tile's V is free only when both
    // chains have read it, so none is more than STAGES + 1 segments ahead.
    uint32_t odd[2][8];
    Board board[kBoard];
    ChunkStarts starts;
    // [chain][half][row]: maxima on the way to the other half of the row, sums at a
    // segment's end.  One buffer is enough: a thread writes the next tile's value only
    // after that tile's S, which is computed only after both halves have released this
    // tile's P, that is, read its values.
    float row[2][2][128];
};
static_assert(sizeof(ChunkShared) <= 3 * 1024, "small arrays");

// Half (h) of one V row of a tile before its first P.V: zeros behind what the unit
// sees, and in place of values that are not finite at positions that not all of its
// rows see (then *odd = seg).  row: its first 128 bytes; the lanes start at different
// 16-byte pieces, against bank conflicts.
template <int KB, bool kF16>
__device__ __noinline__ void fix_v(uint8_t *row, uint32_t h, bool past, volatile uint32_t *odd, uint32_t seg) {
    const uint32_t lane = threadIdx.x & 31;
    constexpr uint32_t em = kF16 ? 0x7c00u : 0x7f80u;
    constexpr int N = KB * 4;  // 16-byte pieces of a half
    auto piece = [&](int u) {
        const uint32_t x = h * N + u;
        return reinterpret_cast<uint4 *>(row + (x >> 3) * BN * 128 + (KB == 2 ? ((x + lane) & 7) : (h * 4 + ((u + lane) & 3))) * 16);
    };
    bool bad = past;
    if (!past)
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const uint4 w = lds128(reinterpret_cast<const uint8_t *>(piece(u)));
            const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) bad |= (ws[e] & em) == em || ((ws[e] >> 16) & em) == em;
        }
    if (!bad) return;
    if (!past) {
        *odd = seg;
        __threadfence_block();  // before the zeros
    }
#pragma unroll 1
    for (int u = 0; u < N; ++u) {
        const uint4 w = past ? make_uint4(0, 0, 0, 0) : *piece(u);
        uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) ws[e] &= ((ws[e] & em) == em ? 0u : 0xffffu) | ((ws[e] >> 16 & em) == em ? 0u : 0xffff0000u);
        *piece(u) = make_uint4(ws[0], ws[1], ws[2], ws[3]);
    }
}

// Barrier over the two warps of 32 rows' halves that also says whether any thread has x.
__device__ __forceinline__ bool pair_any(uint32_t id, bool x) { return group_any(id, 64, x); }

// Infinities and NaN among the V values that row t sees in positions [lo, hi), for 16
// columns.  A weight that is 0 in 32 bits makes NaN of them in a product, and where
// only some rows of the unit see a position they are taken as zeros there.  Weights
// are positive, so such a column is the sum of its values that are not finite.
// odd_from: the first position whose values may have been zeroed (hi or more: none).
// Rare, from global memory, eight positions in flight.
template <bool kF16>
__device__ __noinline__ void add_nonfinite(const TreeParams &p, uint32_t seq, uint32_t head, uint32_t D, uint32_t lo, uint32_t odd_from,
                                           uint32_t hi, uint32_t col, float *o) {
    for (uint32_t c = 0; c < 16; c += 4) {
        const bool nan = o[c] != o[c] || o[c + 1] != o[c + 1] || o[c + 2] != o[c + 2] || o[c + 3] != o[c + 3];
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        for (uint32_t p0 = nan ? lo : max(lo, odd_from); p0 < hi; p0 += 8) {
            float4 v[8];
#pragma unroll
            for (uint32_t u = 0; u < 8; ++u) {
                const uint32_t pos = p0 + u, page = pos < hi ? (uint32_t)tree_table(p, seq)[pos >> p.page_shift] : p.n_pages;
                const size_t row = ((size_t)page << p.page_shift) + (pos & ((1u << p.page_shift) - 1));
                v[u] = page < p.n_pages
                           ? tree_load4<typename std::conditional<kF16, __half, __nv_bfloat16>::type>(p.v, (row * p.n_kv + head) * D + col + c)
                           : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (uint32_t u = 0; u < 8; ++u) {
                const float x[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (!(fabsf(x[e]) < INFINITY)) sum[e] += x[e];
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (sum[e] != 0.f) o[c + e] = nan ? sum[e] : o[c + e] + sum[e];
    }
}

// A wait of the CTA gave up: NaN in the rows of all its segments (in the sums of
// those that the merge joins).  `walk` as at the start.
__device__ __noinline__ void chunk_give_up(const ChunkParams &p, const ChunkStarts *starts, uint32_t D) {
    ChunkWalk walk;
    const ChunkLine line = starts->line;
    walk.line = line;
    ChunkSeg g;
    const uint32_t R = 2 * p.rt;
    for (walk.phase = 0; walk.phase < line.phases; ++walk.phase) {
        walk.begin(p, starts);
        ChunkCut cut = {};
        while (walk.next(p, g)) {
            float *part = g.slot < 2 ? chunk_part(p, D, 2 * walk.piece() + g.slot) : nullptr;
            if (g.slot == 1) cut = chunk_cut(p, line, g);
            for (uint32_t r = threadIdx.x; r < g.rows; r += blockDim.x) {
                if (part) {
                    part[(size_t)R * D + r] = 0.f;
                    part[(size_t)R * (D + 1) + r] = __int_as_float(0x7fffffff);
                } else {
                    uint4 *out = reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p.t.out) + chunk_row(p, g.s.first, g.head, g.row0 + r, D));
                    for (uint32_t u = 0; u < D / 8; ++u) out[u] = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
                }
            }
        }
        if (threadIdx.x == 0) p.cuts[walk.piece()] = cut;
    }
}

template <int D, bool kF16>
__global__ void __launch_bounds__(kThreads, 1) chunk_umma_kernel(const __grid_constant__ ChunkParams cp) {
    using C = CCfg<D>;
    const TreeParams &p = cp.t;
    // 1024-byte alignment for the 128B-swizzle atoms (there is no room for
    // slack; without static shared memory the array starts on such a boundary)
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t *sk_ring = smem + C::OFF_K, *sv_ring = smem + C::OFF_V;
    ChunkShared &sh = *reinterpret_cast<ChunkShared *>(smem + C::OFF_BAR);
    volatile uint32_t *abort_flag = &sh.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < C::STAGES; ++i) {
            mbar_init(&sh.k_full[i], 1);
            mbar_init(&sh.v_full[i], 1);
            mbar_init(&sh.k_empty[i], 2);  // once by each chain, or twice by the one that reads the tile
            mbar_init(&sh.v_empty[i], 2);
        }
        mbar_init(&sh.q_full, 1);
        mbar_init(&sh.q_empty, 2);
        for (int x = 0; x < 2; ++x) {
            mbar_init(&sh.s_full[x], 1);
            mbar_init(&sh.p_full[2 * x], 8);
            mbar_init(&sh.p_full[2 * x + 1], 8);
            mbar_init(&sh.o_final[x], 1);
            mbar_init(&sh.drain[x], 1);
            mbar_init(&sh.turn[x], 1);
        }
        for (uint32_t i = 0; i < kBoard; ++i) {
            mbar_init(&sh.seg_full[i], 1);
            mbar_init(&sh.seg_empty[i], 3 + kSoftmaxWarps);
        }
        sh.abort = 0u;
        fence_mbar_init();
    }
    if (threadIdx.x < 16) sh.odd[threadIdx.x >> 3][threadIdx.x & 7] = 0u;
    if (warp == 0 && lane == 0) {
        prefetch_tmap(&cp.tq);
        prefetch_tmap(&cp.tk);
        prefetch_tmap(&cp.tv);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)),
                     "r"(C::TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (warp == 2) chunk_find(cp, D, &sh.starts);
    __syncthreads();  // the set-up above
    tc_fence_after();
    const uint32_t tmem = *(volatile uint32_t *)&sh.tmem;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the merge may take its place; it waits for this grid

    // The segments in order: every warp sees the same sequence, to its end, also
    // when a wait has given up (then it does no more work for them), so that nobody
    // is left at a barrier.
    uint32_t entry = 0;
    auto segment = [&](Board &b) -> bool {
        uint64_t *seg = &sh.seg_full[entry % kBoard];
        const uint32_t phase = (entry / kBoard) & 1u;
        if (!mbar_test_wait(seg, phase) && !mbar_drain(seg, phase, 8 * p.wait_ns)) {
            *abort_flag = 1u;
            return false;
        }
        __syncwarp();
        const volatile Board *v = &sh.board[entry % kBoard];
        b.seq = v->seq;
        b.first = v->first;
        b.T = v->T;
        b.P = v->P;
        b.head = v->head;
        b.row0 = v->row0;
        b.t0 = v->t0;
        b.n = v->n;
        b.part = v->part;
        return b.n != 0u;
    };
    auto segment_done = [&]() {
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.seg_empty[entry % kBoard]);
        ++entry;
    };

    if (warp == 0 || warp == 2) {
        // ------------------------------------------------------------- producers
        // Warp 0 copies Q and K, warp 2 V.  A lane issues one box: 128-byte
        // column block kb of part `part` of a tile.
        const bool is_k = warp == 0;
        const CUtensorMap *map = is_k ? &cp.tk : &cp.tv;
        uint64_t *full = is_k ? sh.k_full : sh.v_full, *empty = is_k ? sh.k_empty : sh.v_empty;
        uint8_t *ring = is_k ? sk_ring : sv_ring;
        const uint64_t policy = l2_policy_evict_first();
        uint32_t tiles = 0, segs = 0;  // so far
        const uint32_t per_tile = BN / cp.box_rows, part = lane / C::KB, kb = lane % C::KB;
        const uint32_t ps_mask = (1u << p.page_shift) - 1;
        const bool mine = part < per_tile;
        bool live = !(is_k && (p.diag & kTreeStall));
        auto wait_all = [&](uint64_t *bar, uint32_t parity) {
            live = live && __all_sync(0xffffffffu, wait_bar(bar, parity, abort_flag, p.wait_ns));
        };
        auto copy = [&](const Board &b) {
            const uint32_t n = b.n, rows = min(b.T * p.group - b.row0, 2 * cp.rt);
            const bool pair = rows > cp.rt, alone = b.T <= cp.tpg;
            const uint32_t t_end = min(b.T, b.row0 / p.group + cp.tpg);
            const uint32_t lim = b.P < 0 ? 0u : (uint32_t)b.P + t_end;  // positions that the unit sees
            const int32_t *table = tree_table(p, b.seq);
            // Table entries come 32 boxes at a time, one window ahead: lane l
            // holds the first row of box 32 w + l of the segment (-1: past the
            // positions, -2: a page outside the pool).
            auto window = [&](uint32_t w) -> int {
                const uint32_t box = w * 32 + lane, pos = b.t0 * BN + box * cp.box_rows;
                if (box >= n * per_tile || pos >= lim) return -1;
                const uint32_t page = (uint32_t)table[pos >> p.page_shift];
                return page < p.n_pages ? (int)((page << p.page_shift) + (pos & ps_mask)) : -2;
            };
            int win = window(0), win_next = window(1);
            if (is_k) {
                if (segs > 0) wait_all(&sh.q_empty, (segs - 1) & 1u);
                if (!live) return;
                // Q: a box per row tile and column block
                const uint32_t boxes = pair ? 2 * C::KB : C::KB;
                if (lane == 0) mbar_arrive_expect_tx(&sh.q_full, boxes * cp.rt * 128);
                __syncwarp();
                if (lane < boxes) {
                    const uint32_t x = lane / C::KB, c = lane % C::KB;
                    tma_load_3d(smem + x * C::TILE + c * BM * 128, &cp.tq, (int)c * 64, (int)(b.head * p.group),
                                (int)(b.first + (b.row0 + x * cp.rt) / p.group), &sh.q_full);
                }
                __syncwarp();
            }
            for (uint32_t j = 0; j < n && live; ++j, ++tiles) {
                const uint32_t box = j * per_tile, slot = tiles % C::STAGES, use = tiles / C::STAGES;
                if (j > 0 && (box & 31) == 0) {
                    win = win_next;
                    win_next = window(box / 32 + 1);
                }
                int row = __shfl_sync(0xffffffffu, win, (box + part) & 31);
                if (!mine) row = -1;
                if (is_k) {
                    const uint32_t bits = cp.box_rows / 16;  // 16-position blocks of a box
                    uint32_t flag = 0;
                    if (__any_sync(0xffffffffu, row == -2))
                        flag = __reduce_or_sync(0xffffffffu, row == -2 ? ((1u << bits) - 1) << (part * bits) : 0u);
                    if (lane == 0) *(volatile uint32_t *)&sh.bad[tiles % kBadRing] = flag;
                }
                if (use > 0) wait_all(&empty[slot], (use & 1u) ^ 1u);
                if (!live) break;
                const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, row != -1));
                if (lane == 0) mbar_arrive_expect_tx(&full[slot], boxes * cp.box_rows * 128);
                __syncwarp();
                // a page outside the pool is read past the map's end: zeros
                if (row != -1) {
                    uint8_t *dst = ring + slot * C::TILE + kb * BN * 128 + part * cp.box_rows * 128;
                    const int at = row == -2 ? (int)(p.n_pages << p.page_shift) : row;
                    // with one row group K and V are read once
                    if (alone) tma_load_3d_hint(dst, map, (int)kb * 64, (int)b.head, at, &full[slot], policy);
                    else tma_load_3d(dst, map, (int)kb * 64, (int)b.head, at, &full[slot]);
                }
                __syncwarp();
            }
        };
        Board b;
        if (is_k) {
            for (; segment(b); segment_done()) {
                if (live) copy(b);
                ++segs;
            }
        } else {
            const ChunkLine line = sh.starts.line;
            if (lane >= line.phases && lane < cp.most_phases) cp.cuts[lane * gridDim.x + blockIdx.x] = ChunkCut{};
            ChunkWalk walk;
            walk.line = line;
            walk.phase = 0;
            walk.begin(cp, &sh.starts);
            ChunkSeg sg;
            ChunkCut cut = {};
            bool more = true;
            while (more) {
                more = live && !*abort_flag;
                while (more && !walk.next(cp, sg)) {
                    if (lane == 0) cp.cuts[walk.piece()] = cut;
                    cut = {};
                    if (++walk.phase >= line.phases) more = false;
                    else walk.begin(cp, &sh.starts);
                }
                more = __shfl_sync(0xffffffffu, more, 0);
                b = Board{};
                if (more) {
                    b = Board{sg.seq, sg.s.first, sg.s.T, sg.s.P, sg.head, sg.row0, sg.t0, sg.t1 - sg.t0,
                              sg.slot < 2 ? 2 * walk.piece() + sg.slot : kWhole};
                    if (sg.slot == 1) cut = chunk_cut(cp, line, sg);
                }
                // not cut short by the abort flag: the others still read what lies there
                if (entry >= kBoard && !mbar_drain(&sh.seg_empty[entry % kBoard], (entry / kBoard - 1) & 1u, 8 * p.wait_ns)) *abort_flag = 1u;
                __syncwarp();
                if (lane == 0) {
                    sh.board[entry % kBoard] = b;
                    mbar_arrive(&sh.seg_full[entry % kBoard]);
                }
                ++entry;
                __syncwarp();
                if (more && live) copy(b);
            }
        }
        // No copy may outlive the CTA: all have landed unless a wait gave up,
        // and then none is issued any more, so those that have not will soon.
        if (!live) {
            const uint64_t t0 = globaltimer_ns();
            while (globaltimer_ns() - t0 < 1000000ull) {}
        }
        __syncwarp();
    } else if (warp < 4) {
        // ------------------------------------------------------------- MMA issuers
        // The whole warp runs this converged, and one elected lane issues.
        constexpr uint32_t fmt = kF16 ? 0u : 1u;
        constexpr uint32_t idesc_qk = make_idesc(fmt, BM, BN, 0);
        constexpr uint32_t idesc_pv = make_idesc(fmt, BM, D, 1);
        // (from one lane, so that the compiler knows it to be the warp's: operands of
        // tcgen05.mma are uniform registers, and moving them there costs as much as the MMA)
        auto uniform = [](uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); };
        const uint32_t x = uniform((uint32_t)warp >> 1);  // the chain
        const uint64_t dq = smem_desc(smem_u32(smem), 16, 1024);
        const uint64_t dk = smem_desc(smem_u32(sk_ring), 16, 1024);
        const uint64_t dv = smem_desc(smem_u32(sv_ring), BN * 128, 1024);
        const uint32_t s_tmem = uniform(tmem) + x * 128, o_tmem = uniform(tmem) + C::O_COL0 + x * D;
        uint32_t tiles = 0, segs = 0, par = 0;  // tiles and segments so far; phase parity of the P barriers
        bool live = true;
        auto wait_all = [&](uint64_t *bar, uint32_t parity) {
            live = live && __all_sync(0xffffffffu, wait_bar(bar, parity, abort_flag, p.wait_ns));
            tc_fence_after();
            return live;
        };
        uint32_t turns = 0;    // phase parity of this chain's turn
        bool behind = false;   // A: B has a block that follows A's last one
        auto work = [&](bool pair, uint32_t n) {
            const uint32_t nt = pair ? n : (x ? n / 2 : (n + 1) / 2), other = pair ? n : (x ? (n + 1) / 2 : n / 2);
            const uint32_t step = pair ? 1 : 2, j0 = pair ? 0 : x;
            if (!wait_all(&sh.q_full, segs & 1u)) return;
            if (nt == 0) {
                if (elect_one()) mbar_arrive(&sh.q_empty);
                __syncwarp();
                return;
            }
            const uint64_t a_q = dq + (((pair ? x : 0) * C::TILE) >> 4);
            // S from the segment's Q tile and the K tile in a slot: MMAs k0 .. k1 - 1
            auto qk = [&](uint32_t slot, int k0, int k1) {
                const uint64_t b_k = dk + ((slot * C::TILE) >> 4);
#pragma unroll
                for (int kk = k0; kk < k1; ++kk) {
                    const uint32_t off = ((kk >> 2) * (BM * 128) + (kk & 3) * 32) >> 4;
                    tc_mma_ss(s_tmem, a_q + off, b_k + off, idesc_qk, kk > 0);
                }
            };
            // O += P V, step h of the softmax: positions 32 h .. 32 h + 31 of either half
            auto pv = [&](uint32_t slot, int h, bool first) {
                const uint64_t b_v = dv + ((slot * C::TILE) >> 4);
#pragma unroll
                for (int k4 = 0; k4 < 4; ++k4) {
                    const int kk = (k4 >> 1) * 4 + h * 2 + (k4 & 1);
                    tc_mma_ts(o_tmem, s_tmem + kk * 8, b_v + ((kk * 16 * 128) >> 4), idesc_pv, kk > 0 || !first ? 1u : 0u);
                }
            };
            auto qk_done = [&](uint32_t slot, bool last) {
                tc_commit(&sh.s_full[x]);
                tc_commit(&sh.k_empty[slot]);
                if (!pair) tc_commit(&sh.k_empty[slot]);
                if (last) tc_commit(&sh.q_empty);  // this chain has read the segment's Q
            };
            {
                const uint32_t c = tiles + j0, slot = c % C::STAGES;
                if (!wait_all(&sh.k_full[slot], (c / C::STAGES) & 1u)) return;
                if (elect_one()) {
                    qk(slot, 0, D / 16);
                    qk_done(slot, nt == 1);
                }
                __syncwarp();
            }
            for (uint32_t i = 0; i < nt; ++i) {
                // A block: P.V of tile j, and S of the next.  A wait costs this warp 100 to
                // 200 cycles even where nothing is left to wait for, and the tensor core has
                // only one MMA queued: so what is known ahead of P is waited for ahead of it,
                // in one test where that is enough.
                const uint32_t j = j0 + i * step, c = tiles + j, slot = c % C::STAGES, v_par = (c / C::STAGES) & 1u;
                const uint32_t ck = c + step, k_slot = ck % C::STAGES, k_par = (ck / C::STAGES) & 1u;
                const bool more = i + 1 < nt, turn = x || behind;
                bool ahead = !turn || mbar_test_wait(&sh.turn[x], turns);
                if (more) ahead = ahead & mbar_test_wait(&sh.k_full[k_slot], k_par);
                if (i > 0) ahead = ahead & mbar_test_wait(&sh.v_full[slot], v_par);
                if (!__all_sync(0xffffffffu, ahead)) {
                    if (more && !wait_all(&sh.k_full[k_slot], k_par)) return;
                    if (i > 0 && !wait_all(&sh.v_full[slot], v_par)) return;
                    if (turn && !wait_all(&sh.turn[x], turns)) return;
                }
                turns ^= turn;
                if (!wait_all(&sh.p_full[2 * x], par)) return;
                // A segment's first V only after P: P says that both chains are through with
                // the segment before, whose last tiles the slot may have held
                if (i == 0 && !wait_all(&sh.v_full[slot], v_par)) return;
                if (elect_one()) pv(slot, 0, i == 0);
                __syncwarp();
                if (!wait_all(&sh.p_full[2 * x + 1], par)) return;
                if (elect_one()) pv(slot, 1, false);
                __syncwarp();
                par ^= 1u;
                if (elect_one()) {
                    if (more) qk(k_slot, 0, D / 16 - 1);
                    // the other chain's turn, ahead of the last MMA and the commits
                    if (x || i < other) mbar_arrive(&sh.turn[x ^ 1u]);
                    if (more) {
                        qk(k_slot, D / 16 - 1, D / 16);
                        qk_done(k_slot, i + 2 == nt);
                    }
                    tc_commit(&sh.v_empty[slot]);
                    if (!pair) tc_commit(&sh.v_empty[slot]);
                    if (!more) tc_commit(&sh.o_final[x]);
                }
                behind = x == 0 && i < other;
                __syncwarp();
            }
        };
        Board b;
        for (; segment(b); segment_done()) {
            const uint32_t n = uniform(b.n);
            if (live) work(uniform(min(b.T * p.group - b.row0, 2 * cp.rt)) > cp.rt, n);
            tiles += n;
            ++segs;
        }
        if (elect_one()) tc_commit(&sh.drain[x]);  // no MMA outlives the CTA
        __syncwarp();
        mbar_drain(&sh.drain[x], 0, p.wait_ns);
        __syncwarp();
    } else {
        // ------------------------------------------------------------- softmax
        const uint32_t x = (uint32_t)(warp - 4) >> 3, h = (uint32_t)(warp - 4) >> 2 & 1u;
        const uint32_t q4 = warp & 3, r = q4 * 32 + lane, pair_bar = 1 + x * 4 + q4;
        const uint32_t lane_addr = (q4 * 32) << 16;
        const uint32_t s_col = tmem + lane_addr + x * 128;  // P overlays its first 64 columns
        const uint32_t o_base = tmem + lane_addr + C::O_COL0, o_col = o_base + x * D;
        const float c = p.scale_log2;
        uint32_t tiles = 0, done = 0;
        uint32_t finals = 0;  // phase parity of o_final[x]
        Board b;
        for (; segment(b); segment_done()) {
            const uint32_t n = b.n;
            const uint32_t rows = min(b.T * p.group - b.row0, 2 * cp.rt);
            const bool pair = rows > cp.rt;
            const uint32_t nt = pair ? n : (x ? n / 2 : (n + 1) / 2);
            const uint32_t row = (pair ? x * cp.rt : 0) + r;  // row of the group
            const bool valid = r < cp.rt && row < rows;
            const bool warp_live = __any_sync(0xffffffffu, valid);
            const uint32_t t_first = b.row0 / p.group, t_end = min(b.T, t_first + cp.tpg), t = min((b.row0 + row) / p.group, b.T - 1);
            const int32_t sees_all = b.P + (int32_t)t_first;  // the last position that all rows of the unit see
            const int32_t last = b.P + (int32_t)t;            // the last one that this row sees
            const uint32_t kv_first = b.t0 * BN, segs = entry;
            float m_run = -INFINITY, l_run = 0.f;

            for (uint32_t i = 0; i < nt; ++i) {
                const uint32_t j = pair ? i : 2 * i + x;
                const int32_t kv0 = (int32_t)(kv_first + j * BN);
                wait_bar(&sh.s_full[x], (done + i) & 1u, abort_flag, p.wait_ns);
                __syncwarp();
                tc_fence_after();
                const uint32_t bad = *(volatile uint32_t *)&sh.bad[(tiles + j) % kBadRing];
                const bool edge = kv0 + BN - 1 > sees_all;

                if (edge) {
                    // V rows that must not be read as they are: this thread's row is kv0 + r.
                    // In a tile that both chains read each does it before its own P.V, and
                    // what the second one writes is what lies there.
                    const int32_t pos = kv0 + (int32_t)r;
                    const uint32_t cv = tiles + j, slot = cv % C::STAGES;
                    if (__any_sync(0xffffffffu, pos > sees_all)) {
                        wait_bar(&sh.v_full[slot], (cv / C::STAGES) & 1u, abort_flag, p.wait_ns);
                        if (pos > sees_all) fix_v<C::KB, kF16>(sv_ring + slot * C::TILE + r * 128, h, pos >= b.P + (int32_t)t_end, &sh.odd[x][segs & 7u], segs + 1);
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
                const int32_t lim = last - kv0 - (int32_t)h * 64;
                const uint32_t off = bad >> (4 * h);
                const bool masked = edge || bad;
                float sv[64];
                auto mask32 = [&](int q) {  // this half's scores 32 q .. 32 q + 31
                    if (!masked) return;
#pragma unroll
                    for (int k = 32 * q; k < 32 * q + 32; ++k)
                        if (k > lim || (off >> (k / 16) & 1u)) sv[k] = -INFINITY;
                };
                tmem_ld32(s_col + h * 64, sv);
                tmem_ld32(s_col + h * 64 + 32, sv + 32);
                tmem_wait_ld();
                mask32(0);
                mask32(1);
                const float2 c2 = make_float2(c, c);
                float2 nm2, sum2[2];
                uint32_t w[16];
                // P = 2^(s c - m) of 32 scores as packed 16-bit pairs.  All on the SFU: a share
                // of them on the FMA pipe (prefill.cu) costs 5% here, where two threads share
                // a row and the SFU is busy half of the time.
                auto weights = [&](int q) {
#pragma unroll
                    for (int k = 0; k < 32; k += 2) {
                        float2 e = __ffma2_rn(make_float2(sv[q * 32 + k], sv[q * 32 + k + 1]), c2, nm2);
                        e.x = fast_exp2(e.x);
                        e.y = fast_exp2(e.y);
                        sum2[(k >> 1) & 1] = __fadd2_rn(sum2[(k >> 1) & 1], e);
                        w[k >> 1] = pack2<kF16>(e.x, e.y);
                    }
                };
                auto reference = [&]() {
                    const float m_use = (m_run == -INFINITY) ? 0.f : m_run;
                    nm2 = make_float2(-m_use, -m_use);
                    sum2[0] = sum2[1] = make_float2(0.f, 0.f);
                };
                reference();
                float mx4[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float a = fmax3(sv[k], sv[k + 4], sv[k + 8]);
#pragma unroll
                    for (int u = 12; u < 60; u += 8) a = fmax3(a, sv[k + u], sv[k + u + 4]);
                    mx4[k] = fmaxf(a, sv[k + 60]);
                }
                const float mine = fmaxf(fmax3(mx4[0], mx4[1], mx4[2]), mx4[3]) * c;  // c > 0
                // (also in a segment's first tile, which knows no maximum so far: a branch here
                // would keep the two apart, 12% of the long chunk's time)
                weights(0);
                if (pair_any(pair_bar, mine > m_run + kRescaleThreshold)) {
                    sh.row[x][h][r] = mine;
                    named_bar_sync(pair_bar, 64);
                    const float mx = fmaxf(mine, *(volatile float *)&sh.row[x][h ^ 1u][r]);
                    const bool grew = mx > m_run + kRescaleThreshold;
                    const float alpha = !grew ? 1.f : m_run == -INFINITY ? 0.f : fast_exp2(m_run - mx);
                    if (grew) m_run = mx;
                    l_run *= alpha;
                    if (i > 0) {  // this half's columns of O; P.V of the tile before has finished
#pragma unroll 1
                        for (int cc = 0; cc < D / 32; ++cc) {
                            float o[16];
                            tmem_ld16(o_col + h * (D / 2) + cc * 16, o);
                            tmem_wait_ld();
                            uint32_t u[16];
#pragma unroll
                            for (int k = 0; k < 16; ++k) u[k] = __float_as_uint(o[k] * alpha);
                            tmem_st16(o_col + h * (D / 2) + cc * 16, u);
                        }
                    }
                    tmem_ld32(s_col + h * 64, sv);
                    tmem_wait_ld();
                    mask32(0);
                    reference();
                    weights(0);
                }
                // stored over S in two steps, each released to the MMA warp as soon as both
                // halves have written it
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    tmem_st16(s_col + h * 32 + q * 16, w);
                    if (q == 0) weights(1);  // while the first are stored
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.p_full[2 * x + q]);
                }
                const float2 sum = __fadd2_rn(sum2[0], sum2[1]);
                l_run += sum.x + sum.y;
            }
            if (m_run == -INFINITY && l_run == l_run) l_run = 0.f;  // saw nothing (a NaN stays)

            // --------------------------------------------------------- epilogue
            // Row = wa * O_A + wb * O_B, un-normalised, with maximum m and sum l.
            // has_a, has_b: the chain saw something (else its O may be anything).
            float wa = 1.f, wb = 0.f, m = m_run, l = l_run;
            bool has_a = m_run != -INFINITY, has_b = false;
            if (nt > 0) wait_bar(&sh.o_final[x], finals, abort_flag, p.wait_ns);  // the chain's own: its warps meet the other's below
            __syncwarp();
            if (warp_live) {
                // the row's sum of both halves
                sh.row[x][h][r] = l_run;
                named_bar_sync(pair_bar, 64);
                l += *(volatile float *)&sh.row[x][h ^ 1u][r];
                named_bar_sync(pair_bar, 64);  // it has been read
            }
            if (!pair) {
                // one row tile: both chains' (m, l) meet; each of the four threads of a
                // row writes a quarter of the joined row
                if (warp_live) sh.row[x][h][r] = h ? l : m;
                tc_fence_before();
                __syncwarp();
                named_bar_sync(9, kSoftmaxWarps * 32);
                const volatile float *ra = &sh.row[0][0][r];  // [half] 128 apart, [chain] 256
                const float ma = ra[0], la = ra[128], mb = ra[256], lb = ra[384];
                m = fmaxf(ma, mb);
                has_a = ma != -INFINITY;
                has_b = mb != -INFINITY;  // no tiles: -inf
                wa = has_a ? fast_exp2(ma - m) : 0.f;
                wb = has_b ? fast_exp2(mb - m) : 0.f;
                l = wa * la + wb * lb;
                if (la != la || lb != lb) l = la + lb;
            }
            __syncwarp();
            tc_fence_after();
            const float inv = l == 0.f ? 0.f : 1.f / l;
            const size_t at = valid ? chunk_row(cp, b.first, b.head, b.row0 + row, D) : 0;
            float *part = b.part != kWhole ? chunk_part(cp, D, b.part) : nullptr;
            const uint32_t hi = min(kv_first + n * BN, (uint32_t)max(last + 1, 0));
            // either chain: of two that look at the same tile, the second may find zeros
            const bool odd = *(volatile uint32_t *)&sh.odd[0][segs & 7u] == segs + 1 || *(volatile uint32_t *)&sh.odd[1][segs & 7u] == segs + 1;
            if (warp_live) {
                const uint32_t n_cols = pair ? D / 2 : D / 4, first = (pair ? h : 2 * x + h) * n_cols;
                const uint32_t src0 = pair ? o_col : o_base, R = 2 * cp.rt;
#pragma unroll 1
                for (uint32_t col = first; col < first + n_cols; col += 16) {
                    float o[16];
                    __syncwarp();
                    tmem_ld16(src0 + col, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int u = 0; u < 16; ++u) o[u] = has_a ? o[u] * wa : 0.f;
                    if (__any_sync(0xffffffffu, has_b)) {
                        float o2[16];
                        tmem_ld16(o_base + D + col, o2);
                        tmem_wait_ld();
                        if (has_b)
#pragma unroll
                            for (int u = 0; u < 16; ++u) o[u] = fmaf(o2[u], wb, o[u]);
                    }
                    if (valid) {
                        float any[2] = {0.f, 0.f};  // NaN where a column is not finite
#pragma unroll
                        for (int u = 0; u < 16; ++u) any[u & 1] = fmaf(o[u], 0.f, any[u & 1]);
                        if (__builtin_expect((odd || any[0] + any[1] != 0.f) && l == l, 0)) {
                            float tmp[16];  // its address is taken, o's is not
#pragma unroll
                            for (int u = 0; u < 16; ++u) tmp[u] = o[u];
                            add_nonfinite<kF16>(p, b.seq, b.head, D, kv_first, odd ? (uint32_t)max(sees_all + 1, 0) : hi, hi, col, tmp);
#pragma unroll
                            for (int u = 0; u < 16; ++u) o[u] = tmp[u];
                        }
                        if (part) {
                            float4 *dst = reinterpret_cast<float4 *>(part) + (size_t)(col / 4) * R + row;
#pragma unroll
                            for (int u = 0; u < 4; ++u) dst[u * R] = make_float4(o[4 * u], o[4 * u + 1], o[4 * u + 2], o[4 * u + 3]);
                        } else {
                            uint4 *dst = reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p.out) + at + col);
#pragma unroll
                            for (int u = 0; u < 2; ++u)
                                dst[u] = make_uint4(pack2<kF16>(o[8 * u] * inv, o[8 * u + 1] * inv),
                                                    pack2<kF16>(o[8 * u + 2] * inv, o[8 * u + 3] * inv),
                                                    pack2<kF16>(o[8 * u + 4] * inv, o[8 * u + 5] * inv),
                                                    pack2<kF16>(o[8 * u + 6] * inv, o[8 * u + 7] * inv));
                        }
                    }
                }
                if (valid && part && h == 0 && (pair || x == 0)) {
                    part[(size_t)R * D + row] = m;
                    part[(size_t)R * (D + 1) + row] = l;
                }
            }
            tc_fence_before();
            __syncwarp();
            // The next segment's first P.V may overwrite O, and the rows' values be set,
            // once both chains are here.
            if (!pair) named_bar_sync(9, kSoftmaxWarps * 32);
            tiles += n;
            done += nt;
            finals ^= nt > 0;
        }
    }

    tc_fence_before();
    __syncthreads();
    if (*abort_flag) chunk_give_up(cp, &sh.starts, D);
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM_COLS) : "memory");
    }
}

// ---------------------------------------------------------------------------
// Merge of the units that a cut divides: CTA (x, y) serves the one that begins in
// piece x and is divided behind it, and takes its tasks y, y + gridDim.y, ...  A task
// is 8 rows x 32 columns of a warp.  Segments are added in a fixed order, so a result
// does not depend on timing.
// ---------------------------------------------------------------------------
constexpr int kMergeThreads = 256;

template <int D, bool kF16>
__global__ void __launch_bounds__(kMergeThreads) chunk_merge_kernel(const __grid_constant__ ChunkParams cp) {
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the segments' partials are written
    const ChunkCut g = cp.cuts[blockIdx.x];
    const uint32_t from = blockIdx.x, last = g.last;
    const uint32_t R = 2 * cp.rt, tasks = (g.rows + 7) / 8 * (D / 32);
    for (uint32_t task = blockIdx.y * (kMergeThreads / 32) + warp; task < tasks; task += gridDim.y * (kMergeThreads / 32)) {
        const uint32_t row = task / (D / 32) * 8 + (lane & 7), x4 = task % (D / 32) * 8 + (lane >> 3);
        if (row >= g.rows) continue;
        auto part = [&](uint32_t s) { return chunk_part(cp, D, 2 * s + (s == from ? 1u : 0u)); };
        float m = -INFINITY, l = 0.f;
        float4 acc[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
        constexpr uint32_t kBatch = 4;  // segments whose loads are in flight together
        for (uint32_t s0 = from; s0 <= last; s0 += kBatch) {
            float f[kBatch], ls[kBatch];
            float4 y[kBatch][2];
#pragma unroll
            for (uint32_t u = 0; u < kBatch; ++u) {
                const float *src = part(min(s0 + u, last));
                f[u] = src[(size_t)R * D + row];
                ls[u] = src[(size_t)R * (D + 1) + row];
                y[u][0] = reinterpret_cast<const float4 *>(src)[(size_t)x4 * R + row];
                y[u][1] = reinterpret_cast<const float4 *>(src)[(size_t)(x4 + 4) * R + row];
            }
            float mn = m;
#pragma unroll
            for (uint32_t u = 0; u < kBatch; ++u) {
                if (s0 + u > last) f[u] = -INFINITY;
                mn = fmaxf(mn, f[u]);
            }
            const float mu = mn == -INFINITY ? 0.f : mn, old = exp2f(m - mu);  // m -inf: 0
            l *= old;
#pragma unroll
            for (int z = 0; z < 2; ++z) acc[z] = make_float4(acc[z].x * old, acc[z].y * old, acc[z].z * old, acc[z].w * old);
#pragma unroll
            for (uint32_t u = 0; u < kBatch; ++u) {
                if (s0 + u > last) continue;
                const float w = exp2f(f[u] - mu);
                l += w * ls[u];
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                    acc[z].x += w * y[u][z].x;
                    acc[z].y += w * y[u][z].y;
                    acc[z].z += w * y[u][z].z;
                    acc[z].w += w * y[u][z].w;
                }
            }
            m = mn;
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        uint16_t *out = static_cast<uint16_t *>(cp.t.out) + chunk_row(cp, g.first, g.head, g.row0 + row, D) + x4 * 4;
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            const float any = (acc[z].x + acc[z].y) + (acc[z].z + acc[z].w);
            if (__builtin_expect(any != any && l == l, 0)) {
                // a segment's infinity met a weight that is 0 in 32 bits: such a column is
                // the sum of the segments' values that are not finite
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
                for (uint32_t s = from; s <= last; ++s) {
                    const float4 v = reinterpret_cast<const float4 *>(part(s))[(size_t)(x4 + 4 * z) * R + row];
                    const float xs[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!(fabsf(xs[e]) < INFINITY)) sum[e] += xs[e];
                }
                if (sum[0] != 0.f) acc[z].x = sum[0];
                if (sum[1] != 0.f) acc[z].y = sum[1];
                if (sum[2] != 0.f) acc[z].z = sum[2];
                if (sum[3] != 0.f) acc[z].w = sum[3];
            }
            *reinterpret_cast<uint2 *>(out + 16 * z) =
                make_uint2(pack2<kF16>(acc[z].x * inv, acc[z].y * inv), pack2<kF16>(acc[z].z * inv, acc[z].w * inv));
        }
    }
}

// ----------------------------------------------------------------- host
// (d, heads, rows) view of a [rows][heads][d] 16-bit tensor.
bool chunk_map(CUtensorMap *map, const void *base, bool f16, uint32_t d, uint32_t heads, uint64_t rows, uint32_t box_heads,
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
cudaError_t launch_c(const ChunkParams &cp, int num_sms, cudaStream_t st) {
    using C = CCfg<D>;
    auto kern = chunk_umma_kernel<D, kF16>;
    static SmemSet set;  // one for each instantiation
    cudaError_t e = set.allow(kern, C::SMEM);
    if (e != cudaSuccess) return e;
    e = launch_after(kern, dim3(num_sms), kThreads, C::SMEM, st, cp);
    if (e != cudaSuccess || num_sms < 2) return e;
    return launch_after(chunk_merge_kernel<D, kF16>, dim3(num_sms * cp.most_phases - 1, 8), kMergeThreads, 0, st, cp);
}

}  // namespace

// Phases that a batch of so many tokens may take: more need more partial results.
uint32_t chunk_phases(uint64_t n_tokens) { return n_tokens >= 1024 ? kMostPhases : 1; }
size_t chunk_umma_bytes(uint64_t n_tokens, int num_sms) { return sizeof(ChunkCut) * chunk_phases(n_tokens) * num_sms; }

bool chunk_umma_fits(const TreeArgs &a) {
    // positions and tokens are compared in 32 bits with a sign
    return a.p.q_type != BML_F32 && a.p.scale_log2 > 0.f && a.p.group <= (uint32_t)BM && a.p.n_tokens <= 1u << 30;
}

cudaError_t launch_chunk_umma(const TreeArgs &a, int32_t *work, cudaStream_t st) {
    static thread_local ChunkParams cp;
    cp.t = a.p;
    cp.most_phases = chunk_phases(a.p.n_tokens);
    cp.cuts = reinterpret_cast<ChunkCut *>(work);
    const uint32_t group = a.p.group, page = 1u << a.p.page_shift;
    const bool f16 = a.kv_type == BML_F16;
    cp.rt = BM / group * group;
    cp.tpg = 2 * (BM / group);
    cp.box_rows = page < (uint32_t)BN ? page : (uint32_t)BN;
    const uint64_t rows = (uint64_t)a.p.n_pages << a.p.page_shift;
    if (!chunk_map(&cp.tq, a.p.q, f16, a.D, a.p.n_heads, a.p.n_tokens, group, BM / group) ||
        !chunk_map(&cp.tk, a.p.k, f16, a.D, a.p.n_kv, rows, 1, cp.box_rows) ||
        !chunk_map(&cp.tv, a.p.v, f16, a.D, a.p.n_kv, rows, 1, cp.box_rows))
        return cudaErrorInvalidValue;
    if (a.D == 128) return f16 ? launch_c<128, true>(cp, a.num_sms, st) : launch_c<128, false>(cp, a.num_sms, st);
    return f16 ? launch_c<64, true>(cp, a.num_sms, st) : launch_c<64, false>(cp, a.num_sms, st);
}

}  // namespace bml
