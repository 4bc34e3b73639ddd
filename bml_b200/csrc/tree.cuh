// tree.cuh -- attention of drafted tokens over a paged cache: parameters,
// the tile schedule shared by the kernels, and the launch interface.
#pragma once

#include <math.h>

#include <atomic>
#include <type_traits>

#include "paged.cuh"

namespace bml {

constexpr int kTreeTile = 128;         // positions of a schedule tile (tree_umma.cu, tree_warp.cu)
constexpr uint32_t kTreeMaxSeqs = 1024;  // requests of one launch

struct TreeParams {
    const void *q;  // [n_tokens][n_heads][D]
    void *out;      // same shape and type
    const void *k, *v;  // pools [n_pages][page][n_kv][D]
    const int32_t *table;  // [n_seqs][max_pages]
    const int32_t *kv_lens, *node_start;
    const uint64_t *mask;  // [n_tokens][n_words] or null: node t sees nodes 0..t
    uint32_t n_seqs, n_tokens, n_heads, n_kv, group, max_pages, n_pages, page_shift, n_words;
    float scale_log2;
    int q_type;  // bml_dtype of q and out
    // partials: slots of R = hpu * rpg rows, o [D / 4][R][4] un-normalised (a warp
    // whose lanes hold rows writes whole lines), then m [R], l [R]
    float *part;
    uint32_t rpg;        // rows of a row group
    uint32_t hpu;        // kv heads of a unit
    uint32_t tile;       // positions of a schedule tile, a power of two
    uint32_t tile_shift, upr;  // log2(tile); units of a row group: n_kv / hpu (tree_line)
    // a tile's weight: heavy with more rows than heavy_rows, else light
    uint32_t heavy_rows, heavy, light;
    uint32_t lead;  // places ahead of a unit's first tile: what its start and end cost
    uint64_t wait_ns;  // limit of every bounded wait
    uint32_t diag;     // kTreeStall, 0 outside tests
};

// Test-only behaviour (bml_diag_attn_tree): nothing is copied (tree_umma.cu: no
// Q and K), so that the waits for it run out.
constexpr uint32_t kTreeStall = 1u;

struct TreeArgs {
    TreeParams p;
    uint32_t D;
    bml_dtype kv_type;
    // Rows of a request and kv head: on average over the requests with new tokens,
    // and of the widest request (as far as the caller knows; else the average).
    uint32_t rows, widest;
    uint32_t live;  // requests with new tokens, at most
    int num_sms;
    // Whether a form with r rows a row group is for the batch: it fits the average,
    // and reads no request's K and V more than four times (32-bit queries over 16-bit
    // pages: widest is the average, see tree_form).
    bool fits(uint32_t r) const { return rows <= r && widest <= 4 * r; }
    // Tiles of kTreeTile positions of all requests and kv heads, at most: the lengths
    // are on the device, so the tables' width stands for them.
    uint64_t most_tiles() const {
        return (((uint64_t)p.max_pages << p.page_shift) + kTreeTile - 1) / kTreeTile * live * p.n_kv;
    }
    // 32-bit pages: whether row groups of 16 are for the batch, also where they make
    // no more of such tiles than two an SM (see tree_form).
    bool groups16() const { return fits(D == 64 ? 32 : 16) || most_tiles() * ((rows + 15) / 16) <= 2ull * num_sms; }
};
// The kernels: tree.cu, tree_few.cu, tree_warp.cu, tree_umma.cu, tree_umma32.cu.
enum class TreeForm { kF32, kFew, kWarp, kUmma, kUmma32 };
TreeForm tree_form(const TreeArgs &a);

constexpr uint32_t kTreeMaxRows = 256;  // rows of the largest partial slot
cudaError_t launch_tree_merge(const TreeParams &p, uint32_t D, int grid, cudaStream_t st);
size_t tree_workspace_bytes(uint32_t D, int num_sms);

// Allows a kernel its dynamic shared memory, once for each device.
struct SmemSet {
    std::atomic<bool> done[64] = {};
    template <typename F>
    cudaError_t allow(F *kernel, int bytes) {
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        const bool keep = dev >= 0 && dev < 64;
        if (keep && done[dev].load(std::memory_order_acquire)) return cudaSuccess;
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == cudaSuccess && keep) done[dev].store(true, std::memory_order_release);
        return e;
    }
};
cudaError_t launch_tree(const TreeArgs &a, cudaStream_t st);
bool tree_umma_fits(const TreeArgs &a);
cudaError_t launch_tree_warp(const TreeArgs &a, cudaStream_t st);
cudaError_t launch_tree_few(const TreeArgs &a, cudaStream_t st);
cudaError_t launch_tree_umma(const TreeArgs &a, cudaStream_t st);
cudaError_t launch_tree_umma32(const TreeArgs &a, cudaStream_t st);

// Sets what follows from the other fields, and says whether the schedule can
// count the launch's tiles in 32 bits, whatever the lengths on the device are.
inline uint64_t tree_most_units(const TreeParams &p) {
    return ((uint64_t)p.n_tokens * p.group / p.rpg + p.n_seqs) * p.upr;
}
inline bool tree_line(TreeParams &p) {
    p.tile_shift = 0;
    while (1u << p.tile_shift < p.tile) ++p.tile_shift;
    p.upr = p.n_kv / p.hpu;
    const uint64_t tiles = (((uint64_t)p.max_pages << p.page_shift) + p.tile - 1) / p.tile;
    return tree_most_units(p) * p.heavy <= 0xffffffffull / (tiles + p.lead);
}

#ifdef __CUDACC__
// ---------------------------------------------------------------------------
// Schedule.  A unit is one (request, hpu kv heads, row group): for each of the
// heads the query rows (node t, q head g of the kv head) of up to rpg
// consecutive t * group + g, over all positions of the request.  Units are laid
// out request by request, heads by heads, row group by row group, each as its
// number of tiles of positions times a tile's weight, with `lead` places ahead of
// the first tile, and the line of all places is cut evenly over the CTAs,
// so the lengths stay on the GPU and no CTA works longer than another by more
// than a tile.  A unit that a cut divides leaves partial results (max, sum,
// un-normalised output) which tree_merge_kernel joins in tile order.
// ---------------------------------------------------------------------------
struct TreeSeq {
    uint32_t first;  // first token row
    uint32_t T, L;   // drafted tokens; positions (0: refused, its rows are zero)
    uint32_t rows, groups, tiles;
    uint32_t w_last, weight;  // a tile's weight in the last row group; in all groups of a head
    uint32_t places;          // of a head
};

// A tile's weight in a row group.  kW false: all are 1 (the kernels without
// weights leave them out, since a launch meets this code cold).
template <bool kW>
__device__ __forceinline__ uint32_t tree_weight(const TreeParams &p, uint32_t rows) {
    return !kW ? 1u : rows > p.heavy_rows ? p.heavy : p.light;
}

// What the device holds of a request: rows [a, b), positions.
struct TreeRaw {
    int32_t a, b, L;
};
// kEarly: before griddepcontrol.wait (the merge, which reads past L1).
template <bool kEarly>
__device__ __forceinline__ TreeRaw tree_raw(const TreeParams &p, uint32_t i) {
    if (kEarly) return {__ldcg(p.node_start + i), __ldcg(p.node_start + i + 1), __ldcg(p.kv_lens + i)};
    return {p.node_start[i], p.node_start[i + 1], p.kv_lens[i]};
}
template <bool kW>
__device__ __forceinline__ TreeSeq tree_seq(const TreeParams &p, const TreeRaw &raw) {
    TreeSeq s;
    const int32_t a = raw.a, b = raw.b, L = raw.L;
    const bool rows_ok = a >= 0 && b > a && (uint32_t)b <= p.n_tokens;
    s.first = rows_ok ? (uint32_t)a : 0u;
    s.T = rows_ok ? (uint32_t)(b - a) : 0u;
    const uint32_t most = p.mask ? p.n_words * 64 : kTreeMaxNodes;
    const bool ok = s.T <= most && L >= (int32_t)s.T && (uint64_t)L <= ((uint64_t)p.max_pages << p.page_shift);
    s.L = ok ? (uint32_t)L : 0u;
    s.rows = s.T * p.group;
    s.groups = (s.rows + p.rpg - 1) / p.rpg;
    s.tiles = s.L ? (s.L + p.tile - 1) >> p.tile_shift : 1u;
    s.w_last = tree_weight<kW>(p, s.rows - (s.groups - 1) * p.rpg);
    s.weight = s.groups ? (s.groups - 1) * tree_weight<kW>(p, p.rpg) + s.w_last : 0u;
    s.places = s.weight * s.tiles + s.groups * p.lead;
    return s;
}

template <bool kEarly, bool kW>
__device__ __forceinline__ TreeSeq tree_seq(const TreeParams &p, uint32_t i) {
    return tree_seq<kW>(p, tree_raw<kEarly>(p, i));
}

struct TreeShared {
    uint32_t warp_sums[32], warp_units[32];
    uint32_t base;  // place of seq's first tile on the line
    uint32_t seq, unit;
};

// How a line of weight `total` is cut for up to `grid` CTAs, at least a heavy
// tile's weight each: the first `more` take one more than the others.  A tile
// belongs to the CTA in whose part it begins; a part inside one unit holds at
// least one beginning.
template <bool kW>
struct TreeCuts {
    uint32_t each, more, active;
    __device__ __forceinline__ TreeCuts(const TreeParams &p, uint32_t total, uint32_t grid) {
        const uint32_t most = kW ? total / p.heavy : total;
        active = most < 1 ? (total ? 1u : 0u) : most < grid ? most : grid;
        each = active ? total / active : 0u;
        more = total - each * active;
    }
    __device__ __forceinline__ uint32_t at(uint32_t b) const { return each * b + min(b, more); }
    // the CTA that holds place w
    __device__ __forceinline__ uint32_t owner(uint32_t w) const {
        const uint32_t wide = more * (each + 1);
        return w < wide ? w / (each + 1) : more + (w - wide) / each;
    }
};

// CTA b's range of the line, and where it starts.
struct TreeRange {
    uint32_t w0, w1, base, total;
    uint32_t seq;
    TreeSeq s;  // of seq
};

// The request that holds tile w (by_unit: unit w) of the line.  Up to 128
// requests every warp finds it by itself (four requests a lane, no barrier);
// with more the CTA's threads share them.  Every thread of the CTA calls it.
struct TreePlace {
    uint32_t total, units;  // of the line
    uint32_t seq, base, unit0;  // the request, its first tile, its first unit
    TreeSeq s;
};

template <bool kEarly, bool kW, typename Target>
__device__ __forceinline__ TreePlace tree_find(const TreeParams &p, TreeShared *sh, bool by_unit, Target target) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, upr = p.upr;
    const bool alone = p.n_seqs <= 128;
    const uint32_t members = alone ? 32u : blockDim.x, me = alone ? lane : threadIdx.x;
    const uint32_t per = (p.n_seqs + members - 1) / members;
    const uint32_t i0 = min(me * per, p.n_seqs), i1 = min(i0 + per, p.n_seqs);
    uint32_t tiles = 0, units = 0;
    uint32_t n4[4] = {0, 0, 0, 0}, t4[4] = {0, 0, 0, 0};  // alone: units and tiles of the lane's requests
    TreeRaw raw[4] = {};
    if (alone) {
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k)
            if (i0 + k < i1) {
                raw[k] = tree_raw<kEarly>(p, i0 + k);
                const TreeSeq s = tree_seq<kW>(p, raw[k]);
                n4[k] = s.groups * upr;
                t4[k] = upr * s.places;
                units += n4[k];
                tiles += t4[k];
            }
    } else {
        for (uint32_t i = i0; i < i1; ++i) {
            const TreeSeq s = tree_seq<kEarly, kW>(p, i);
            units += s.groups * upr;
            tiles += upr * s.places;
        }
    }
    uint32_t inc_t = tiles, inc_u = units;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t a = __shfl_up_sync(0xffffffffu, inc_t, o), b = __shfl_up_sync(0xffffffffu, inc_u, o);
        if (lane >= (uint32_t)o) {
            inc_t += a;
            inc_u += b;
        }
    }
    TreePlace r;
    uint32_t ft = inc_t - tiles, fu = inc_u - units;
    if (alone) {
        r.total = __shfl_sync(0xffffffffu, inc_t, 31);
        r.units = __shfl_sync(0xffffffffu, inc_u, 31);
    } else {
        if (lane == 31) {
            sh->warp_sums[warp] = inc_t;
            sh->warp_units[warp] = inc_u;
        }
        __syncthreads();
        r.total = r.units = 0;
        for (uint32_t w = 0; w < blockDim.x / 32; ++w) {
            if (w < warp) {
                ft += sh->warp_sums[w];
                fu += sh->warp_units[w];
            }
            r.total += sh->warp_sums[w];
            r.units += sh->warp_units[w];
        }
    }
    const uint32_t w = target(r.total);
    const bool mine = by_unit ? w >= fu && w < fu + units : w >= ft && w < ft + tiles;
    uint32_t seq = i0;
    if (alone) {
#pragma unroll
        for (uint32_t k = 0; k < 3; ++k)
            if (mine && seq == i0 + k && (by_unit ? w >= fu + n4[k] : w >= ft + t4[k])) {
                fu += n4[k];
                ft += t4[k];
                raw[0] = raw[k + 1];  // of seq
                ++seq;
            }
        const uint32_t who = __ffs(__ballot_sync(0xffffffffu, mine)) - 1;  // none: lane 31's, unused
        r.seq = __shfl_sync(0xffffffffu, seq, who & 31);
        r.base = __shfl_sync(0xffffffffu, ft, who & 31);
        r.unit0 = __shfl_sync(0xffffffffu, fu, who & 31);
        r.s = tree_seq<kW>(p, TreeRaw{__shfl_sync(0xffffffffu, raw[0].a, who & 31), __shfl_sync(0xffffffffu, raw[0].b, who & 31),
                                  __shfl_sync(0xffffffffu, raw[0].L, who & 31)});
    } else {
        if (mine) {
            while (true) {
                const TreeSeq s = tree_seq<kEarly, kW>(p, seq);
                const uint32_t n = s.groups * upr, t = upr * s.places;
                if ((by_unit ? w < fu + n : w < ft + t) || seq + 1 >= i1) break;
                fu += n;
                ft += t;
                ++seq;
            }
            sh->seq = seq;
            sh->base = ft;
            sh->unit = fu;
        }
        __syncthreads();
        r.seq = sh->seq;
        r.base = sh->base;
        r.unit0 = sh->unit;
        if (r.seq < p.n_seqs) r.s = tree_seq<kEarly, kW>(p, r.seq);
    }
    return r;
}

// CTA b's range.  w0 == w1: nothing for this CTA.
template <bool kW, bool kEarly = false>
__device__ __forceinline__ TreeRange tree_range(const TreeParams &p, TreeShared *sh, uint32_t b, uint32_t grid) {
    TreeRange r;
    r.w0 = r.w1 = 0;
    const TreePlace at = tree_find<kEarly, kW>(p, sh, false, [&](uint32_t total) {
        const TreeCuts<kW> cuts(p, total, grid);
        if (b < cuts.active) {
            r.w0 = cuts.at(b);
            r.w1 = cuts.at(b + 1);
        }
        return r.w0;
    });
    r.total = at.total;
    r.base = at.base;
    r.seq = at.seq;
    r.s = at.s;
    return r;
}

// A unit's place on the line: its tiles lie at [u0, u0 + w * s.tiles).
struct TreeUnit {
    uint32_t u0, w, total;
    uint32_t seq, head, rg;
    TreeSeq s;
    bool found;
};

// The unit with index u in line order (for the merge).
__device__ __forceinline__ TreeUnit tree_unit(const TreeParams &p, TreeShared *sh, uint32_t u) {
    const TreePlace at = tree_find<true, true>(p, sh, true, [&](uint32_t) { return u; });
    TreeUnit r = {};
    r.found = u < at.units;
    r.total = at.total;
    if (r.found) {
        r.seq = at.seq;
        r.s = at.s;
        const uint32_t in = u - at.unit0;
        r.head = in / r.s.groups;
        r.rg = in - r.head * r.s.groups;
        r.u0 = at.base + r.head * r.s.places + r.rg * (tree_weight<true>(p, p.rpg) * r.s.tiles + p.lead) + p.lead;
        r.w = r.rg + 1 == r.s.groups ? r.s.w_last : tree_weight<true>(p, p.rpg);
        r.head *= p.hpu;
    }
    return r;
}

// The segments of a range in order: consecutive tiles of one unit.
struct TreeSeg {
    uint32_t seq, head, rg;  // head: the first of the unit's
    uint32_t t0, t1;     // tiles of the unit, [t0, t1)
    uint32_t u0, w;      // the unit's place on the line, a tile's weight
    uint32_t row0, rows; // first row (t * group + g) and row count of the group
    uint32_t slot;       // partial slot of the CTA: 0 the unit began before this range, 1 it ends after it, 2 whole
    TreeSeq s;
};

template <bool kW>
struct TreeWalk {
    uint32_t pos, end, base;
    uint32_t seq;
    TreeSeq s;
    __device__ __forceinline__ explicit TreeWalk(const TreeRange &r) : pos(r.w0), end(r.w1), base(r.base), seq(r.seq), s(r.s) {}
    template <bool kEarly = false>
    __device__ __forceinline__ bool next(const TreeParams &p, TreeSeg &g) {
        while (pos < end) {
            uint32_t per_head;
            while (pos - base >= (per_head = s.places) * p.upr) {
                base += per_head * p.upr;
                if (++seq >= p.n_seqs) {  // only with a node_start that does not ascend
                    pos = end;
                    return false;
                }
                s = tree_seq<kEarly, kW>(p, seq);
            }
            const uint32_t off = pos - base, wf = tree_weight<kW>(p, p.rpg);
            const uint32_t head = off / per_head, in_head = off - head * per_head;
            const uint32_t full = wf * s.tiles + p.lead;
            g.rg = s.groups > 1 ? min(in_head / full, s.groups - 1) : 0u;
            g.w = g.rg + 1 == s.groups ? s.w_last : wf;
            const uint32_t in = in_head - g.rg * full, left = end - pos;
            const uint32_t out = min(in + left, g.w * s.tiles + p.lead);  // where the range ends in the unit
            const uint32_t ti = max(in, p.lead) - p.lead, to = max(out, p.lead) - p.lead;
            g.t0 = kW ? (ti + g.w - 1) / g.w : ti;
            g.t1 = kW ? (to + g.w - 1) / g.w : to;
            g.u0 = pos - in + p.lead;
            pos += out - in;
            if (g.t0 == g.t1) continue;  // no tile begins here
            g.seq = seq;
            g.s = s;
            g.head = head * p.hpu;
            g.row0 = g.rg * p.rpg;
            g.rows = min(p.rpg, s.rows - g.row0);
            g.slot = g.t0 > 0 ? 0u : (g.t1 < s.tiles ? 1u : 2u);
            return true;
        }
        return false;
    }
};

// Floats of a partial slot, a multiple of 4: slots start on 16 bytes also where
// the rows are odd in number (125 of them for groups of 5).
__device__ __forceinline__ size_t tree_slot(const TreeParams &p, uint32_t D) { return ((size_t)p.rpg * p.hpu * (D + 2) + 3) & ~(size_t)3; }
// Partial slot `which` (0 or 1) of CTA b.
__device__ __forceinline__ float *tree_part(const TreeParams &p, uint32_t D, uint32_t b, uint32_t which) {
    return p.part + (2 * (size_t)b + which) * tree_slot(p, D);
}

// Element index of row r (t * group + g) of the unit's kv head `h` in q and out.
__device__ __forceinline__ size_t tree_row(const TreeParams &p, const TreeSeg &g, uint32_t r, uint32_t D, uint32_t h = 0) {
    const uint32_t t = r / p.group, qg = r - t * p.group;
    return ((size_t)(g.s.first + t) * p.n_heads + (size_t)(g.head + h) * p.group + qg) * D;
}

// A wait of the CTA gave up: NaN in the rows of all its segments (in the sums of
// those that the merge joins), which covers segments that nobody has begun.
// Out of line, for every thread of the CTA; 16-bit results.
template <bool kW>
__device__ __noinline__ void tree_give_up(const TreeParams &p, TreeShared *sh, uint32_t D) {
    const TreeRange range = tree_range<kW>(p, sh, blockIdx.x, gridDim.x);
    TreeWalk<kW> walk(range);
    TreeSeg g;
    while (walk.next(p, g)) {
        const uint32_t R = p.rpg * p.hpu;
        float *part = g.slot < 2 ? tree_part(p, D, blockIdx.x, g.slot) : nullptr;
        for (uint32_t i = threadIdx.x; i < g.rows * p.hpu; i += blockDim.x) {
            const uint32_t h = i / g.rows, r = i - h * g.rows;
            if (part) {
                part[(size_t)R * D + h * p.rpg + r] = 0.f;
                part[(size_t)R * (D + 1) + h * p.rpg + r] = __int_as_float(0x7fffffff);
            } else {
                uint4 *out = reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p.out) + tree_row(p, g, g.row0 + r, D, h));
                for (uint32_t u = 0; u < D / 8; ++u) out[u] = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
            }
        }
    }
}

// Whether node t of a request sees position pos >= P (= node pos - P).
__device__ __forceinline__ bool tree_sees(const TreeParams &p, const TreeSeq &s, uint32_t t, uint32_t node) {
    if (node >= s.T) return false;
    if (!p.mask) return node <= t;
    return (p.mask[(size_t)(s.first + t) * p.n_words + (node >> 6)] >> (node & 63)) & 1;
}

// Which of the nodes n0 .. n0 + 15 (n0 > -16; below 0: committed positions,
// seen by all) node t of a request sees.
__device__ __forceinline__ uint32_t tree_see16(const TreeParams &p, const TreeSeq &s, uint32_t t, int32_t n0) {
    if (n0 >= (int32_t)s.T) return 0u;
    const uint32_t first = n0 < 0 ? 0u : (uint32_t)n0, left = s.T - first;
    uint64_t w;  // bit i: node first + i
    if (p.mask) {
        const uint64_t *m = p.mask + (size_t)(s.first + t) * p.n_words;
        const uint32_t i = first >> 6, b = first & 63;
        w = m[i] >> b;
        if (b > 48 && i + 1 < p.n_words) w |= m[i + 1] << (64 - b);
    } else {
        const int32_t k = (int32_t)t - (int32_t)first;  // nodes up to t
        w = k < 0 ? 0ull : k >= 63 ? ~0ull : (2ull << k) - 1;
    }
    if (left < 16) w &= (1ull << left) - 1;
    return n0 < 0 ? (uint32_t)(w << -n0) | ((1u << -n0) - 1) : (uint32_t)w;
}

// hi: x rounded to TF32's 10 fraction bits, half away from zero, with integer
// operations (a conversion instruction runs at a quarter of their rate and set
// tree_f32_kernel's time: 4 requests of 618 to 2671 positions 85 -> 75 us).  lo: the rest, of
// which the matrix unit takes the upper bits itself.  For softmax weights: x at
// most 2^8, or NaN (which lo keeps).
__device__ __forceinline__ void tf32_split(float x, uint32_t &hi, uint32_t &lo) {
    hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
    lo = __float_as_uint(x - __uint_as_float(hi));
}
// A value of any size.  hi stays finite: of a value that would round to infinity,
// of an infinity and of a NaN it is the largest TF32 value of their sign, and lo
// is the rest (an infinity or NaN as such), so that x * inf is what it should be
// and not x * inf - x * inf.
__device__ __forceinline__ void tf32_split_any(float x, uint32_t &hi, uint32_t &lo) {
    float h = __uint_as_float((__float_as_uint(x) + 0x1000u) & 0xffffe000u);
    asm("min.xorsign.abs.f32 %0, %0, 0f7F7FE000;" : "+f"(h));  // the smaller magnitude, the sign of h
    hi = __float_as_uint(h);
    lo = __float_as_uint(x - h);
}

template <bool kF16>
__device__ __forceinline__ bool odd16(uint16_t x) {  // not finite
    constexpr uint16_t em = kF16 ? 0x7c00u : 0x7f80u;
    return (x & em) == em;
}
template <bool kF16>
__device__ __forceinline__ float wide16(uint16_t x) {
    return kF16 ? __half2float(*reinterpret_cast<const __half *>(&x)) : __uint_as_float((uint32_t)x << 16);
}

// x as TERMS 16-bit terms, the largest first: x is their sum to 24 (three
// bf16) or 22 bits (two f16).  f16's smallest step is 2^-24, so its second term
// is kept kTermScale times as large: 22 bits down to 2^-14, and a step of 2^-36
// below that (2^-24 without).
template <bool kF16>
constexpr float kTermScale = kF16 ? 4096.f : 1.f;
template <bool kF16, int TERMS>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t (&t)[TERMS]) {
#pragma unroll
    for (int i = 0; i < TERMS; ++i) {
        t[i] = pack2<kF16>(x, y);
        if (i + 1 < TERMS) {
            x = (x - wide16<kF16>((uint16_t)t[i])) * kTermScale<kF16>;
            y = (y - wide16<kF16>((uint16_t)(t[i] >> 16))) * kTermScale<kF16>;
        }
    }
}

// Four values of a pool row.
template <typename KT>
__device__ __forceinline__ float4 tree_load4(const void *pool, size_t at) {
    if constexpr (sizeof(KT) == 4) {
        return *reinterpret_cast<const float4 *>(static_cast<const float *>(pool) + at);
    } else {
        const uint2 w = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(pool) + at);
        if constexpr (std::is_same<KT, __half>::value) {
            const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&w.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&w.y));
            return make_float4(a.x, a.y, b.x, b.y);
        }
        return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                           __uint_as_float(w.y & 0xffff0000u));
    }
}

// Positions [lo, hi) of a request's kv head, and the node of the row that looks.
struct TreeSpan {
    uint32_t seq, head, t, lo, hi;
    TreeSeq s;
};

// Infinities and NaN among the V values that a row sees.  In products a weight
// that is 0 in 32 bits, or a split weight's lower term, makes NaN of them; those of
// drafted nodes, which other rows do not see, are taken as zeros there.  So a
// column that came out NaN though the row's sum of weights is a number, and all
// columns where a node's values were zeroed, are looked up here: weights are
// positive, so such a column is the sum of its values that are not finite.
// o: n columns from `col` on, un-normalised; nan: some of them are NaN (else only
// the end of the request is looked at, and added).  Rare, from global memory.
template <int D, typename KT>
__device__ __noinline__ void tree_nonfinite(const TreeParams &p, const TreeSpan &a, uint32_t col, uint32_t n, bool nan, float *o) {
    // tree_f32_kernel zeroes in whole blocks, of up to 32 positions: some before the
    // nodes, and what is not finite may be added twice
    const uint32_t P = a.s.L - min(a.s.T, a.s.L), begin = nan ? a.lo : max(a.lo, P - min(P, 32u)), end = min(a.hi, a.s.L);
    for (uint32_t c = 0; c < n; c += 4) {
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        for (uint32_t pos = begin; pos < end; ++pos) {
            if (pos >= P && !tree_sees(p, a.s, a.t, pos - P)) continue;
            const uint32_t page = (uint32_t)p.table[(size_t)a.seq * p.max_pages + (pos >> p.page_shift)];
            if (page >= p.n_pages) continue;
            const size_t row = ((size_t)page << p.page_shift) + (pos & ((1u << p.page_shift) - 1));
            const float4 v = tree_load4<KT>(p.v, (row * p.n_kv + a.head) * D + col + c);
            const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (!(fabsf(x[e]) < INFINITY)) sum[e] += x[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (sum[e] != 0.f) o[c + e] = nan ? sum[e] : o[c + e] + sum[e];
    }
}
// For four columns, where they need it.  l: the row's sum of weights; odd: the
// segment has a node with zeroed values.
template <int D, typename KT>
__device__ __forceinline__ void tree_nonfinite4(const TreeParams &p, const TreeSeg &g, uint32_t head, uint32_t row, uint32_t col, float l,
                                                bool odd, float4 &x) {
    const float any = (x.x + x.y) + (x.z + x.w);  // inf - inf: looked up for nothing
    if (__builtin_expect((odd || any != any) && l == l, 0)) {
        const TreeSpan a = {g.seq, head, (g.row0 + row) / p.group, g.t0 << p.tile_shift, g.t1 << p.tile_shift, g.s};
        float o[4] = {x.x, x.y, x.z, x.w};
        tree_nonfinite<D, KT>(p, a, col, 4, any != any, o);
        x = make_float4(o[0], o[1], o[2], o[3]);
    }
}

// 16 bytes global -> shared; bytes = 0 writes zeros and reads nothing.
__device__ __forceinline__ void cp16(uint32_t dst, const void *src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Barrier over `threads` threads that also says whether any of them has x.
__device__ __forceinline__ bool group_any(uint32_t id, uint32_t threads, bool x) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred a, b;\n\t"
        "setp.ne.u32 a, %1, 0;\n\t"
        "bar.red.or.pred b, %2, %3, a;\n\t"
        "selp.u32 %0, 1, 0, b;\n\t}"
        : "=r"(r)
        : "r"((uint32_t)x), "r"(id), "r"(threads)
        : "memory");
    return r != 0;
}
// A warp's sum of weights l >= 0 on the way to its CTA's join, with a sign that
// says whether a drafted node's V values that are not finite were taken as zeros.
__device__ __forceinline__ float odd_sign(float l, bool odd) { return odd ? -l : l; }
__device__ __forceinline__ bool sign_odd(float l) { return __float_as_uint(l) >> 31; }
#endif

}  // namespace bml
