// pages.cu -- a paged cache's pages shared, returned and moved: requests that
// continue another's positions, requests that end or are rolled back, and the
// pool packed to its front.  No reference counterpart (one flat buffer a layer,
// crates/compiler/src/kv_cache.rs:25-181 in SugarFreeDoNoSo/bml).
//
// shared[page] counts a page's holders beyond the first, so that page_plan, whose
// new pages have one holder, needs to know nothing of it.  Counts, tables and
// the free list are small: one cluster of CTAs does the bookkeeping of a call,
// with a cluster barrier where one step needs all of the one before.  Results
// do not depend on the order of atomics: they add and subtract integers, and
// nothing reads a count before its barrier.
#include <cooperative_groups.h>

#include "pages.cuh"

namespace cg = cooperative_groups;

namespace bml {

namespace {

constexpr uint32_t kBook = 8;  // CTAs of the bookkeeping cluster
constexpr int kThreads = 512;
constexpr int kFreeThreads = 1024;
// From so many pages, or entries of the free list, on a release goes over all SMs.  512
// requests, 131,000 pages: 43 us by the cluster, 10.4 over all SMs; 32,768 pages 12.3 and
// 7.6; 16,384 9.2 and 7.3; 4096 7.7 and 6.8.  But four launches take the host 11.5 us,
// one 5.7.
constexpr uint32_t kWidePages = 16384;

// Block-wide exclusive sum; every thread gets the total.  sums: one per warp.
__device__ __forceinline__ uint32_t block_before(uint32_t x, uint32_t *sums, uint32_t *total) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    uint32_t inc = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t a = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= (uint32_t)o) inc += a;
    }
    if (lane == 31) sums[warp] = inc;
    __syncthreads();
    uint32_t before = 0, all = 0;
    for (uint32_t w = 0; w < nw; ++w) {
        if (w < warp) before += sums[w];
        all += sums[w];
    }
    __syncthreads();
    *total = all;
    return before + inc - x;
}

__device__ __forceinline__ uint32_t block_sum(uint32_t x, uint32_t *sums) {
    uint32_t total;
    block_before(x, sums, &total);
    return total;
}

// Every CTA's value of x, by rank, in the caller's `all` (shared memory of its own
// for each use, so that one cluster barrier is enough).
__device__ __forceinline__ void cluster_gather(cg::cluster_group &cl, uint32_t x, uint32_t *all) {
    if (threadIdx.x < cl.num_blocks()) *cl.map_shared_rank(all + cl.block_rank(), threadIdx.x) = x;
    cl.sync();
}

// bytes from src to dst by the whole CTA, eight units a thread in flight.
template <typename U>
__device__ __forceinline__ void copy_cta(char *dst, const char *src, uint32_t bytes) {
    constexpr uint32_t kAtOnce = 8;
    const U *s = reinterpret_cast<const U *>(src);
    U *d = reinterpret_cast<U *>(dst);
    const uint32_t units = bytes / sizeof(U);
    for (uint32_t i0 = threadIdx.x; i0 < units; i0 += blockDim.x * kAtOnce) {
        U x[kAtOnce];
#pragma unroll
        for (uint32_t k = 0; k < kAtOnce; ++k)
            if (i0 + k * blockDim.x < units) x[k] = __ldcs(s + i0 + k * blockDim.x);
#pragma unroll
        for (uint32_t k = 0; k < kAtOnce; ++k)
            if (i0 + k * blockDim.x < units) __stcs(d + i0 + k * blockDim.x, x[k]);
    }
}

// ---------------------------------------------------------------------------
// page_fork
//
// Fork j: row dst_j of the tables continues row src_j, len = lens[src_j]:
//   pages 0 .. len / page - 1 are full: table[dst][k] = table[src][k], shared += 1;
//   a part-filled page is copied (its len % page rows, all layers) to
//   free[used + (part-filled pages of the forks before)], since both requests
//   will write behind their rows.
// Every CTA redoes the plan (a few loads a fork, one scan); cluster 0 keeps the
// books, and all copy.  Memory-bound in the copies: 48 forks, 32 layers, rows of 2 KB
// 81 us (6.2 TB/s; four CTAs an SM: 87 with one, 97 with two); 8 forks of one prompt 7 us,
// launch and the plan's dependent loads; in a pool of 131,000 pages 12.8, whose counts one
// cluster copies.
// ---------------------------------------------------------------------------
struct ForkOne {
    int32_t len;       // positions; -1: refused
    int32_t fresh;     // page that takes the part-filled one, -1: none
};

template <typename U>
__global__ void __launch_bounds__(kThreads) page_fork_kernel(const __grid_constant__ ForkParams p) {
    extern __shared__ int32_t sh[];
    ForkOne *one = reinterpret_cast<ForkOne *>(sh);  // [m]
    int32_t *claim = sh + 2 * p.m;                   // [n]: the first fork into the row
    __shared__ uint32_t sums[kThreads / 32], s_granted;
    cg::cluster_group cl = cg::this_cluster();
    const uint32_t ps = 1u << p.pool.page_shift;
    for (uint32_t i = threadIdx.x; i < p.n; i += kThreads) claim[i] = 0x7fffffff;
    if (threadIdx.x == 0) s_granted = 0;
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (uint32_t j = threadIdx.x; j < p.m; j += kThreads)
        if ((uint32_t)p.dst[j] < p.n) atomicMin(&claim[p.dst[j]], (int32_t)j);
    __syncthreads();
    const uint32_t used = (uint32_t)min(max(*p.free_used, 0), (int32_t)p.n_free);
    uint32_t cum = 0;  // part-filled pages of the forks before this round of threads
    for (uint32_t j0 = 0; j0 < p.m; j0 += kThreads) {
        const uint32_t j = j0 + threadIdx.x;
        int32_t st = 0, len = 0, need = 0;
        if (j < p.m) {
            const uint32_t s = (uint32_t)p.src[j], d = (uint32_t)p.dst[j];
            if (s >= p.n || d >= p.n || claim[d] != (int32_t)j || p.owned[d] != 0 || p.lens[d] != 0) st = kPlanBad;
            else {
                len = p.lens[s];
                need = len < 0 ? 0 : (int32_t)(((int64_t)len + ps - 1) >> p.pool.page_shift);
                if (len < 0 || p.owned[s] < need || need > (int32_t)p.max_pages) st = kPlanBad;
            }
        }
        const uint32_t part = j < p.m && st == 0 && (len & (ps - 1)) ? 1 : 0;
        uint32_t total;
        const uint32_t before = cum + block_before(part, sums, &total);
        cum += total;
        if (part && before + 1 > p.n_free - used) st = kPlanNoPages;
        if (part && st == 0) atomicMax(&s_granted, before + 1);
        if (j < p.m) {
            one[j] = {st ? -1 : len, part && st == 0 ? p.free_pages[used + before] : -1};
            if (blockIdx.x == 0) p.status[j] = st;
        }
    }
    __syncthreads();

    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (blockIdx.x < kBook) {
        const uint32_t rank = cl.block_rank(), me = rank * kThreads + threadIdx.x, all = kBook * kThreads;
        if (me == 0) *p.free_used_out = (int32_t)(used + s_granted);
        for (uint32_t i = me; i < p.n; i += all) {
            const int32_t j = claim[i] == 0x7fffffff ? -1 : claim[i], len = j >= 0 ? one[j].len : -1;
            p.lens_out[i] = len >= 0 ? len : p.lens[i];
            p.owned_out[i] = len >= 0 ? (int32_t)(((int64_t)len + ps - 1) >> p.pool.page_shift) : p.owned[i];
        }
        for (uint32_t i = me; i < p.pool.n_pages; i += all) p.shared_out[i] = p.shared[i];
        cl.sync();
        for (uint32_t j = rank * (kThreads / 32) + warp; j < p.m; j += kBook * (kThreads / 32)) {
            if (one[j].len < 0) continue;
            const uint32_t s = (uint32_t)p.src[j], d = (uint32_t)p.dst[j], full = (uint32_t)one[j].len >> p.pool.page_shift;
            if (s == d) continue;  // an idle row onto itself
            const int32_t *from = p.table + (size_t)s * p.max_pages;
            int32_t *to = p.table + (size_t)d * p.max_pages;
            for (uint32_t k = lane; k < full; k += 32) {
                const int32_t page = from[k];
                to[k] = page;
                if ((uint32_t)page < p.pool.n_pages) atomicAdd(&p.shared_out[page], 1);
            }
            if (lane == 0 && one[j].fresh >= 0) to[full] = one[j].fresh;
        }
    }

    // copies: an item is a (fork, layer, K or V), in an order that spreads the forks
    const uint64_t per = 2ull * p.pool.n_layers, items = per * p.m;
    for (uint64_t it = blockIdx.x; it < items; it += gridDim.x) {
        const uint32_t j = (uint32_t)(it / per), lw = (uint32_t)(it - j * per);
        if (one[j].fresh < 0) continue;
        const uint32_t len = (uint32_t)one[j].len, rows = len & (ps - 1);
        const uint32_t from = (uint32_t)p.table[(size_t)p.src[j] * p.max_pages + (len >> p.pool.page_shift)], to = (uint32_t)one[j].fresh;
        if (from >= p.pool.n_pages || to >= p.pool.n_pages || from == to) continue;
        char *base = ((lw & 1) ? p.pool.v_pool : p.pool.k_pool) + (lw >> 1) * p.pool.layer_bytes;
        const uint64_t page_bytes = (uint64_t)p.pool.row_bytes << p.pool.page_shift;
        copy_cta<U>(base + to * page_bytes, base + from * page_bytes, rows * p.pool.row_bytes);
    }
}

// ---------------------------------------------------------------------------
// page_free
//
// Request i keeps len' = min(len, keep) positions (keep < 0: everything, its spare
// pages too) and its first ceil(len' / page) pages.  A page is gone when as many
// rows release it as hold it (shared + 1).  The taken part of the free list,
// free[0 .. used), is partitioned: the pages still held, then the gone ones, each
// in the order they had, and used ends between them.
// ---------------------------------------------------------------------------
struct FreeOne {
    int32_t len, stay, owned, status;
};
__device__ __forceinline__ FreeOne free_one(const FreeParams &p, uint32_t i) {
    FreeOne r = {p.lens[i], 0, p.owned[i], 0};
    const int32_t keep = p.keep[i], ps = 1 << p.page_shift;
    r.stay = r.owned;
    if (keep < 0 || r.len < 0 || r.owned < 0 || r.owned > (int32_t)p.max_pages) return r;
    const int32_t len = min(r.len, keep), whole = len >> p.page_shift;
    if (len < r.len && (len & (ps - 1)) && whole < r.owned) {
        // ends inside a page: the request will write there, which other holders must not see
        const uint32_t page = (uint32_t)p.table[(size_t)i * p.max_pages + whole];
        if (page < p.n_pages && p.shared[page] > 0) {
            r.status = kPageShared;
            return r;
        }
    }
    r.len = len;
    r.stay = min(r.owned, whole + ((len & (ps - 1)) ? 1 : 0));
    return r;
}

// Independent loads of a loop's next kAtOnce elements, so that they are in flight
// together (131,000 pages, 512 requests: 71 us with one at a time).
constexpr uint32_t kAtOnce = 4;

__global__ void __launch_bounds__(kFreeThreads) page_free_kernel(const __grid_constant__ FreeParams p) {
    __shared__ uint32_t sums[kFreeThreads / 32], s_gone[kBook];
    cg::cluster_group cl = cg::this_cluster();
    const uint32_t rank = cl.block_rank(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t me = rank * kFreeThreads + threadIdx.x, all = kBook * kFreeThreads;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t used = (uint32_t)min(max(*p.free_used, 0), (int32_t)p.n_free);
    auto copy = [&](const int32_t *from, int32_t *to, uint32_t first, uint32_t end, int32_t least) {
        for (uint32_t i0 = first + me; i0 < end; i0 += all * kAtOnce) {
            int32_t x[kAtOnce];
#pragma unroll
            for (uint32_t k = 0; k < kAtOnce; ++k)
                if (i0 + k * all < end) x[k] = from[i0 + k * all];
#pragma unroll
            for (uint32_t k = 0; k < kAtOnce; ++k)
                if (i0 + k * all < end) to[i0 + k * all] = max(x[k], least);
        }
    };
    copy(p.shared, p.shared_out, 0, p.n_pages, 0);
    for (uint32_t i = me; i < p.n; i += all) {
        const FreeOne r = free_one(p, i);
        p.lens_out[i] = r.len;
        p.owned_out[i] = r.stay;
        p.status[i] = r.status;
    }
    copy(p.free_pages, p.free_out, used, p.n_free, INT32_MIN);
    cl.sync();
    for (uint32_t i = rank * (kFreeThreads / 32) + warp; i < p.n; i += kBook * (kFreeThreads / 32)) {
        const int32_t stay = __ldcg(p.owned_out + i), owned = p.owned[i];
        const uint32_t drop = stay < owned ? (uint32_t)(owned - stay) : 0u;  // then owned is at most max_pages
        const int32_t *row = p.table + (size_t)i * p.max_pages + stay;
        for (uint32_t k0 = lane; k0 < drop; k0 += 32 * kAtOnce) {
            uint32_t page[kAtOnce];
#pragma unroll
            for (uint32_t k = 0; k < kAtOnce; ++k) page[k] = k0 + 32 * k < drop ? (uint32_t)row[k0 + 32 * k] : 0xffffffffu;
#pragma unroll
            for (uint32_t k = 0; k < kAtOnce; ++k)
                if (page[k] < p.n_pages) atomicSub(&p.shared_out[page[k]], 1);
        }
    }
    cl.sync();
    // a run of the taken part for each thread: its gone pages counted, then both kinds placed
    const uint32_t run = (used + all - 1) / all, a = min(me * run, used), b = min(a + run, used);
    uint32_t mine = 0;
    int32_t page[kAtOnce];
    bool gone[kAtOnce];
    auto look = [&](uint32_t i0) {
#pragma unroll
        for (uint32_t k = 0; k < kAtOnce; ++k) page[k] = i0 + k < b ? p.free_pages[i0 + k] : -1;
#pragma unroll
        for (uint32_t k = 0; k < kAtOnce; ++k) gone[k] = (uint32_t)page[k] < p.n_pages && __ldcg(&p.shared_out[page[k]]) < 0;
    };
    for (uint32_t i0 = a; i0 < b; i0 += kAtOnce) {
        look(i0);
#pragma unroll
        for (uint32_t k = 0; k < kAtOnce; ++k) mine += i0 + k < b && gone[k];
    }
    uint32_t cta;
    uint32_t before = block_before(mine, sums, &cta);
    cluster_gather(cl, cta, s_gone);
    uint32_t total = 0;
    for (uint32_t r = 0; r < kBook; ++r) {
        if (r < rank) before += s_gone[r];
        total += s_gone[r];
    }
    const uint32_t left = used - total;
    if (me == 0) *p.free_used_out = (int32_t)left;
    for (uint32_t i0 = a; i0 < b; i0 += kAtOnce) {
        if (run > kAtOnce) look(i0);  // else as it is
#pragma unroll
        for (uint32_t k = 0; k < kAtOnce; ++k)
            if (i0 + k < b) {
                p.free_out[gone[k] ? left + before : i0 + k - before] = page[k];
                before += gone[k];
            }
    }
    cl.sync();  // every flag has been read
    for (uint32_t i0 = me; i0 < p.n_pages; i0 += all * kAtOnce) {
        int32_t x[kAtOnce];
#pragma unroll
        for (uint32_t k = 0; k < kAtOnce; ++k) x[k] = i0 + k * all < p.n_pages ? __ldcg(&p.shared_out[i0 + k * all]) : 0;
#pragma unroll
        for (uint32_t k = 0; k < kAtOnce; ++k)
            if (x[k] < 0) p.shared_out[i0 + k * all] = 0;
    }
}

// The same over all SMs for long lists: a launch a step in place of a cluster barrier.
// work: the gone pages of each tile of the taken part, then a bit for each entry, so
// that the last step need not look a page up while another CTA clears it.
constexpr int kWideThreads = 256;
struct FreeTile {
    uint32_t a, b, used;
    __device__ __forceinline__ explicit FreeTile(const FreeParams &p) {
        used = (uint32_t)min(max(*p.free_used, 0), (int32_t)p.n_free);
        a = (uint32_t)min((uint64_t)blockIdx.x * p.tile, (uint64_t)used);
        b = (uint32_t)min((uint64_t)a + p.tile, (uint64_t)used);
    }
};

__global__ void __launch_bounds__(kWideThreads) free_start_kernel(const __grid_constant__ FreeParams p) {
    const uint32_t me = blockIdx.x * kWideThreads + threadIdx.x, all = gridDim.x * kWideThreads;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t used = (uint32_t)min(max(*p.free_used, 0), (int32_t)p.n_free);
    for (uint32_t i = me; i < p.n_pages; i += all) p.shared_out[i] = max(p.shared[i], 0);
    for (uint64_t i = (uint64_t)used + me; i < p.n_free; i += all) p.free_out[i] = p.free_pages[i];
    for (uint32_t i = me; i < p.n; i += all) {
        const FreeOne r = free_one(p, i);
        p.lens_out[i] = r.len;
        p.owned_out[i] = r.stay;
        p.status[i] = r.status;
    }
}

__global__ void __launch_bounds__(kWideThreads) free_release_kernel(const __grid_constant__ FreeParams p) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t i = blockIdx.x;
    const int32_t stay = p.owned_out[i], owned = p.owned[i];
    const uint32_t drop = stay < owned ? (uint32_t)(owned - stay) : 0u;  // then owned is at most max_pages
    const int32_t *row = p.table + (size_t)i * p.max_pages + stay;
    for (uint32_t k = threadIdx.x; k < drop; k += kWideThreads) {
        const uint32_t page = (uint32_t)row[k];
        if (page < p.n_pages) atomicSub(&p.shared_out[page], 1);
    }
}

__global__ void __launch_bounds__(kWideThreads) free_count_kernel(const __grid_constant__ FreeParams p) {
    __shared__ uint32_t sums[kWideThreads / 32];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const FreeTile t(p);
    uint32_t mine = 0;
    for (uint32_t i0 = t.a; i0 < t.b; i0 += kWideThreads) {
        const uint32_t i = i0 + threadIdx.x, page = i < t.b ? (uint32_t)p.free_pages[i] : 0xffffffffu;
        const uint32_t word = __ballot_sync(0xffffffffu, page < p.n_pages && p.shared_out[page] < 0);
        if ((threadIdx.x & 31) == 0 && i < t.b) {
            p.work[kFreeTiles + i / 32] = word;
            mine += __popc(word);
        }
    }
    mine = block_sum(mine, sums);
    if (threadIdx.x == 0) p.work[blockIdx.x] = mine;
}

__global__ void __launch_bounds__(kWideThreads) free_place_kernel(const __grid_constant__ FreeParams p) {
    __shared__ uint32_t sums[kWideThreads / 32];
    const uint32_t lane = threadIdx.x & 31, me = blockIdx.x * kWideThreads + threadIdx.x, all = gridDim.x * kWideThreads;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const FreeTile t(p);
    uint32_t before = 0, total = 0;
    for (uint32_t i = threadIdx.x; i < gridDim.x; i += kWideThreads) {
        const uint32_t x = p.work[i];
        total += x;
        if (i < blockIdx.x) before += x;
    }
    total = block_sum(total, sums);
    before = block_sum(before, sums);
    const uint32_t left = t.used - total;
    if (me == 0) *p.free_used_out = (int32_t)left;
    for (uint32_t i0 = t.a; i0 < t.b; i0 += kWideThreads) {
        const uint32_t i = i0 + threadIdx.x, word = i < t.b ? p.work[kFreeTiles + i / 32] : 0u;
        uint32_t some;
        const uint32_t warps = block_before(lane == 0 ? __popc(word) : 0u, sums, &some);  // lane 0: of the warps before
        const uint32_t at = before + __shfl_sync(0xffffffffu, warps, 0) + __popc(word & ((1u << lane) - 1));
        if (i < t.b) p.free_out[(word >> lane & 1u) ? left + at : i - at] = p.free_pages[i];
        before += some;
    }
    for (uint32_t i = me; i < p.n_pages; i += all)
        if (p.shared_out[i] < 0) p.shared_out[i] = 0;
}

// ---------------------------------------------------------------------------
// page_compact
//
// With H held pages, those at H and behind move into the pages below H that nobody
// holds, both in ascending order; sources and destinations are disjoint, so the
// moves need no order.  Tables and shared counts follow the pages, and the free
// list becomes 0, 1, 2, ... with H taken.  The first kernel finds the moves, the
// second makes them.  Memory-bound: 32 requests, 32 layers, pages of 131 KB 551 us (6.1
// TB/s); 200 pages of 131,000 moved in one layer 76 us, the first kernel's five walks of the pool.
// work: where[n_pages] (mark, then a page's new place), from[n_pages], to[n_pages],
// the number of moves.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(kThreads) page_moves_kernel(const __grid_constant__ CompactParams p) {
    __shared__ uint32_t sums[kThreads / 32], s_live[kBook], s_move[kBook], s_hole[kBook];
    cg::cluster_group cl = cg::this_cluster();
    const uint32_t rank = cl.block_rank(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = p.pool.n_pages;
    const uint32_t me = rank * kThreads + threadIdx.x, all = kBook * kThreads;
    int32_t *where = p.work, *from = where + n, *to = from + n;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (uint32_t i = me; i < n; i += all) {
        where[i] = 0;
        p.free_out[i] = (int32_t)i;
    }
    cl.sync();
    for (uint32_t i = rank * (kThreads / 32) + warp; i < p.n; i += kBook * (kThreads / 32)) {
        const int32_t own = min(p.owned[i], (int32_t)p.max_pages);
        for (int32_t k = (int32_t)lane; k < own; k += 32) {
            const uint32_t page = (uint32_t)p.table[(size_t)i * p.max_pages + k];
            if (page < n) where[page] = 1;
        }
    }
    cl.sync();
    const uint32_t run = (n + kBook - 1) / kBook, a = min(rank * run, n), b = min(a + run, n);
    uint32_t live = 0;
    for (uint32_t i = a + threadIdx.x; i < b; i += kThreads) live += __ldcg(&where[i]) != 0;
    live = block_sum(live, sums);
    cluster_gather(cl, live, s_live);
    uint32_t held = 0;
    for (uint32_t r = 0; r < kBook; ++r) held += s_live[r];
    uint32_t move = 0, hole = 0;
    for (uint32_t i = a + threadIdx.x; i < b; i += kThreads) {
        const bool w = __ldcg(&where[i]) != 0;
        move += w && i >= held;
        hole += !w && i < held;
    }
    move = block_sum(move, sums);
    hole = block_sum(hole, sums);
    cluster_gather(cl, move, s_move);
    cluster_gather(cl, hole, s_hole);
    uint32_t m0 = 0, h0 = 0, moves = 0;
    for (uint32_t r = 0; r < kBook; ++r) {
        if (r < rank) {
            m0 += s_move[r];
            h0 += s_hole[r];
        }
        moves += s_move[r];
    }
    if (me == 0) {
        *p.free_used_out = (int32_t)held;
        to[n] = (int32_t)moves;
    }
    const uint32_t move0 = m0;
    for (uint32_t i0 = a; i0 < b; i0 += kThreads) {
        const uint32_t i = i0 + threadIdx.x;
        const bool w = i < b && __ldcg(&where[i]) != 0, mv = w && i >= held, ho = i < b && !w && i < held;
        uint32_t some;
        const uint32_t at = block_before((uint32_t)mv | (uint32_t)ho << 16, sums, &some);  // at most 512 of each
        if (mv) from[m0 + (at & 0xffff)] = (int32_t)i;
        if (ho) to[h0 + (at >> 16)] = (int32_t)i;
        m0 += some & 0xffff;
        h0 += some >> 16;
    }
    cl.sync();
    m0 = move0;
    for (uint32_t i0 = a; i0 < b; i0 += kThreads) {
        const uint32_t i = i0 + threadIdx.x;
        const bool w = i < b && __ldcg(&where[i]) != 0, mv = w && i >= held;
        uint32_t some;
        const uint32_t at = m0 + block_before(mv, sums, &some);
        const int32_t place = mv ? __ldcg(&to[at]) : (int32_t)i;
        if (w) p.shared_out[place] = p.shared[i];
        if (i < b) {
            where[i] = place;
            if (i >= held) p.shared_out[i] = 0;
        }
        m0 += some;
    }
}

// Pages from[m] to to[m], in all layers, K and V.  A CTA copies a unit a thread of a
// page (a piece) at a time, kInFlight pieces in flight.
template <typename U, typename I>
__device__ __forceinline__ void move_pages(const PoolParams &p, const I *from, const I *to, uint32_t moves) {
    constexpr uint32_t kInFlight = 8;
    const uint64_t page_bytes = (uint64_t)p.row_bytes << p.page_shift;  // below 2^31
    const uint32_t units = (uint32_t)(page_bytes / sizeof(U)), pieces = (units + kThreads - 1) / kThreads, both = 2 * p.n_layers;
    // (move, layer and side, piece) as digits, advanced by the grid's
    const uint32_t dp = gridDim.x % pieces, dl = gridDim.x / pieces % both, dm = gridDim.x / pieces / both;
    uint32_t at = blockIdx.x % pieces, lw = blockIdx.x / pieces % both, m = blockIdx.x / pieces / both;
    while (m < moves) {
        U x[kInFlight], *d[kInFlight];
#pragma unroll
        for (uint32_t k = 0; k < kInFlight; ++k) {
            const uint32_t u = at * kThreads + threadIdx.x;
            d[k] = nullptr;
            if (m < moves && u < units) {
                char *base = ((lw & 1) ? p.v_pool : p.k_pool) + (lw >> 1) * p.layer_bytes;
                d[k] = reinterpret_cast<U *>(base + (uint32_t)to[m] * page_bytes) + u;
                x[k] = __ldcs(reinterpret_cast<const U *>(base + (uint32_t)from[m] * page_bytes) + u);
            }
            at += dp;
            lw += dl + (at >= pieces);
            at -= at >= pieces ? pieces : 0;
            m += dm + (lw >= both);
            lw -= lw >= both ? both : 0;
        }
#pragma unroll
        for (uint32_t k = 0; k < kInFlight; ++k)
            if (d[k]) __stcs(d[k], x[k]);
    }
}

template <typename U>
__global__ void __launch_bounds__(kThreads) page_move_kernel(const __grid_constant__ CompactParams p) {
    const uint32_t n = p.pool.n_pages;
    const int32_t *where = p.work, *from = where + n, *to = from + n;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint64_t entries = (uint64_t)p.n * p.max_pages;
    for (uint64_t e = (uint64_t)blockIdx.x * kThreads + threadIdx.x; e < entries; e += (uint64_t)gridDim.x * kThreads) {
        const uint32_t i = (uint32_t)(e / p.max_pages), k = (uint32_t)(e - (uint64_t)i * p.max_pages);
        const int32_t page = p.table[e];
        p.table_out[e] = (int32_t)k < p.owned[i] && (uint32_t)page < n ? where[page] : page;
    }
    move_pages<U>(p.pool, from, to, (uint32_t)to[n]);
}

// Both in one launch for a small pool: every CTA finds all the moves, from bits in
// shared memory, and makes its share of them.  6 requests of 16 pages in 200, 22 layers:
// 7.8 us, 14.7 in two launches; 32 of 60 in 4000, 4 layers 22.7 and 31.5; 128 of 32 in
// 8192, one layer 15.1 and 22.3.  A CTA an SM: its search costs more than its copies gain
// from more of them (the first case with two 10.0 us, with four 13.7).
constexpr uint32_t kSmallPages = 8192, kSmallEntries = 16384;

template <typename U>
__global__ void __launch_bounds__(kThreads) page_compact_kernel(const __grid_constant__ CompactParams p) {
    constexpr uint32_t kWords = kSmallPages / 32, kAtOnce = 8;
    static_assert(kWords <= kThreads, "a word a thread");  // and 16-bit page numbers
    __shared__ uint32_t held_bits[kWords], before[kWords], sums[kThreads / 32];
    __shared__ uint16_t from[kSmallPages / 2], to[kSmallPages / 2];  // as many movers as holes below them
    const uint32_t n = p.pool.n_pages, tid = threadIdx.x, me = blockIdx.x * kThreads + tid, all = gridDim.x * kThreads;
    const uint32_t entries = p.n * p.max_pages;
    if (tid < kWords) held_bits[tid] = 0;
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    auto held_entry = [&](uint32_t e) { return (int32_t)(e % p.max_pages) < p.owned[e / p.max_pages]; };
    for (uint32_t e0 = tid; e0 < entries; e0 += kThreads * kAtOnce) {
        uint32_t page[kAtOnce];
#pragma unroll
        for (uint32_t k = 0; k < kAtOnce; ++k) {
            const uint32_t e = e0 + k * kThreads;
            page[k] = e < entries && held_entry(e) ? (uint32_t)p.table[e] : 0xffffffffu;
        }
#pragma unroll
        for (uint32_t k = 0; k < kAtOnce; ++k)
            if (page[k] < n) atomicOr(&held_bits[page[k] >> 5], 1u << (page[k] & 31));
    }
    __syncthreads();
    const uint32_t word = tid < kWords ? held_bits[tid] : 0u;
    uint32_t held;
    const uint32_t first = block_before(__popc(word), sums, &held);  // held pages before this word
    if (tid < kWords) before[tid] = first;
    __syncthreads();
    // pages below i that are held
    auto rank = [&](uint32_t i) { return before[i >> 5] + __popc(held_bits[i >> 5] & ((1u << (i & 31)) - 1)); };
    const uint32_t stay = held < n ? rank(held) : held;  // held pages below H; H is n only if all are
    const uint32_t moves = held - stay;
    for (uint32_t i = tid; i < n; i += kThreads) {
        const bool h = held_bits[i >> 5] >> (i & 31) & 1u;
        if (h && i >= held) from[rank(i) - stay] = (uint16_t)i;
        if (!h && i < held) to[i - rank(i)] = (uint16_t)i;
    }
    __syncthreads();

    for (uint32_t e = me; e < entries; e += all) {
        const int32_t page = p.table[e];
        int32_t place = page;
        if ((uint32_t)page < n && (uint32_t)page >= held && held_entry(e)) place = to[rank((uint32_t)page) - stay];
        p.table_out[e] = place;
    }
    for (uint32_t i = me; i < n; i += all) {
        p.free_out[i] = (int32_t)i;
        if (held_bits[i >> 5] >> (i & 31) & 1u) p.shared_out[i < held ? i : to[rank(i) - stay]] = p.shared[i];
        if (i >= held) p.shared_out[i] = 0;
    }
    if (me == 0) *p.free_used_out = (int32_t)held;
    move_pages<U>(p.pool, from, to, moves);
}

bool wide(const PoolParams &p) {
    return p.row_bytes % 16 == 0 && ((reinterpret_cast<uintptr_t>(p.k_pool) | reinterpret_cast<uintptr_t>(p.v_pool)) & 15u) == 0;
}

}  // namespace

cudaError_t launch_page_fork(const ForkParams &p, cudaStream_t st) {
    const int smem = (int)(p.m * sizeof(ForkOne) + p.n * sizeof(int32_t));  // at most 48 KB (kPlanMaxSeqs of both)
    const uint64_t items = 2ull * p.pool.n_layers * p.m, most = (uint64_t)p.num_sms * 4;
    uint32_t grid = (uint32_t)(items < most ? items : most);
    grid = grid < kBook ? kBook : (grid + kBook - 1) / kBook * kBook;
    auto kern = wide(p.pool) ? page_fork_kernel<uint4> : page_fork_kernel<uint16_t>;
    if (smem > 47 * 1024) {  // with the static part above what needs no allowance
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 64 * 1024);
        if (e != cudaSuccess) return e;
    }
    return launch_clusters(kern, kBook, dim3(grid), kThreads, smem, st, p);
}

cudaError_t launch_page_free(const FreeParams &p, cudaStream_t st) {
    if (p.n_pages < kWidePages && p.n_free < kWidePages)
        return launch_clusters(page_free_kernel, kBook, dim3(kBook), kFreeThreads, 0, st, p);
    FreeParams q = p;
    q.tile = (p.n_free + kFreeTiles - 1) / kFreeTiles;  // in whole words of the bits
    q.tile = q.tile < kWideThreads ? kWideThreads : (q.tile + 31) / 32 * 32;
    const uint32_t tiles = (p.n_free + q.tile - 1) / q.tile, grid = tiles < kFreeTiles / 4 ? kFreeTiles / 4 : tiles;
    cudaError_t e = launch_after(free_start_kernel, dim3((uint32_t)p.num_sms * 2), kWideThreads, 0, st, q);
    if (e == cudaSuccess) e = launch_after(free_release_kernel, dim3(p.n), kWideThreads, 0, st, q);
    if (e == cudaSuccess) e = launch_after(free_count_kernel, dim3(grid), kWideThreads, 0, st, q);
    if (e == cudaSuccess) e = launch_after(free_place_kernel, dim3(grid), kWideThreads, 0, st, q);
    return e;
}

cudaError_t launch_page_compact(const CompactParams &p, cudaStream_t st) {
    const bool w = wide(p.pool);
    if (p.pool.n_pages <= kSmallPages && (uint64_t)p.n * p.max_pages <= kSmallEntries)
        return launch_after(w ? page_compact_kernel<uint4> : page_compact_kernel<uint16_t>, dim3((uint32_t)p.num_sms), kThreads, 0, st, p);
    const cudaError_t e = launch_clusters(page_moves_kernel, kBook, dim3(kBook), kThreads, 0, st, p);
    if (e != cudaSuccess) return e;
    return launch_after(w ? page_move_kernel<uint4> : page_move_kernel<uint16_t>, dim3((uint32_t)p.num_sms * 4), kThreads, 0, st, p);
}

}  // namespace bml
