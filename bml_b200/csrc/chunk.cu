// chunk.cu -- attention of chunks of any number of new tokens over a paged cache,
// where chunk_umma.cu does not take them: 32-bit queries, a scale of 0, groups of
// more than 128 q heads, and batches of few tokens.
//
// Row t of a request's T new tokens sees the positions 0 .. P + t, P = L - T.  A
// chunk is cut into pieces of W consecutive tokens: piece k is a request of its
// own, W tokens behind P + k W positions on the same row of the block table, and
// the kernels of drafted tokens (tree*.cu) compute it.  W * group is at most 256
// rows (W = 1 for larger groups), so the masked part of a piece is at most W
// positions wide; its K and V are read once for each of its row groups, whose size
// is the kernel's (128 rows at most with 32-bit queries).  How many pieces a batch has is on
// the device; n_seqs + n_tokens / W bound it, and those that are none have no tokens.
#include "tree.cuh"

namespace bml {

namespace {

constexpr int kThreads = 1024;
constexpr uint32_t kPieceRows = 256;
// 32-bit queries over 16-bit pages: tree_umma32.cu from so many rows a request or piece
// on (on average).  3 requests of 706 fresh tokens, d = 128, group 4: 163 us, 271 with
// tree_warp.cu; 8 of 64 tokens behind 1000: 88 and 131; 32 of 16 behind 2000: 222 and
// 220, of 8: 217 and 128.
constexpr uint32_t kTf32Rows = 80;
// Batches of so few tokens are a call of tree*.cu as they are, no request having more
// than such a call takes: no pieces are made (32-bit queries: 3 us less), and with
// 16-bit queries those kernels start sooner than chunk_umma.cu (behind 1000 positions,
// bf16, d = 128: one token 11.9 us, 15.3 there; 64 tokens 18.9 and 25.2; one request of
// 128 24.7 and 28.2; f16, d = 64: 8 of one token 9.6 and 16.0, one of 128 20.0 and 22.5).
// The start that they save is the same behind any number of positions, and a tile of
// 64 tokens costs more there: 8 of 64 tokens 48.2 and 34.7, 3 of 80 31.3 and 28.1, 64
// tokens of one among 64 idle requests 37.3 and 26.0 (d = 64: 21.3 and 20.1).  For more than
// 8 requests of a token each they would be the faster ones (32 of one: 28.2 and 38.4, d = 64
// 16.0 and 22.6): tree_attention is the call for such a batch.
constexpr uint32_t kFewTokens = 64, kFewSeqs = 8;

struct PieceParams {
    const int32_t *node_start, *kv_lens;  // [n + 1], [n]
    uint32_t n, n_tokens, width, most;    // width: tokens of a piece; most: pieces
    uint64_t room;                        // positions of a row of the block table
    int32_t *first;                       // [n + 1]: a request's first piece
    int32_t *start, *end, *lens, *row_of;  // [most] each: the pieces.  An end of its own: behind
                                           // a request there may be rows that nobody computes
};

// One CTA: pieces of each request, their prefix sums, then a piece a thread.
__global__ void __launch_bounds__(kThreads) chunk_pieces_kernel(const PieceParams p) {
    __shared__ uint32_t sums[kThreads / 32];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    auto tokens = [&](uint32_t i) -> uint32_t {
        const int32_t a = p.node_start[i], b = p.node_start[i + 1];
        return a >= 0 && b > a && (uint32_t)b <= p.n_tokens ? (uint32_t)(b - a) : 0u;
    };
    uint32_t base = 0;
    for (uint32_t i0 = 0; i0 < p.n; i0 += kThreads) {
        const uint32_t i = i0 + threadIdx.x, x = i < p.n ? (tokens(i) + p.width - 1) / p.width : 0u;
        uint32_t inc = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= (uint32_t)o) inc += y;
        }
        if (lane == 31) sums[warp] = inc;
        __syncthreads();
        uint32_t before = 0, all = 0;
        for (uint32_t w = 0; w < kThreads / 32; ++w) {
            if (w < warp) before += sums[w];
            all += sums[w];
        }
        if (i < p.n) p.first[i] = (int32_t)min(base + before + inc - x, p.most);
        base = min(base + all, p.most);  // more only with a node_start that does not ascend
        __syncthreads();
    }
    if (threadIdx.x == 0) p.first[p.n] = (int32_t)base;
    __syncthreads();
    for (uint32_t v = threadIdx.x; v < p.most; v += kThreads) {
        int32_t start = 0, end = 0, len = 0;
        uint32_t row = 0;
        if (v < base) {
            uint32_t lo = 0, hi = p.n;  // the last request whose first piece is at most v
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) >> 1;
                if ((uint32_t)p.first[mid] <= v) lo = mid;
                else hi = mid;
            }
            const uint32_t T = tokens(lo), k = (v - (uint32_t)p.first[lo]) * p.width;
            const int32_t L = p.kv_lens[lo];
            row = lo;
            start = p.node_start[lo] + (int32_t)min(k, T);
            end = p.node_start[lo] + (int32_t)min(k + p.width, T);
            // a refused request, or one whose positions its row does not hold: none
            if (L >= (int32_t)T && (uint64_t)L <= p.room) len = L - (int32_t)T + (int32_t)min(k + p.width, T);
        }
        p.start[v] = start;
        p.end[v] = end;
        p.lens[v] = len;
        p.row_of[v] = (int32_t)row;
    }
}

}  // namespace

size_t chunk_work_bytes(uint64_t n_tokens, uint64_t n_seqs, int num_sms) {
    // pieces of one token at the least (groups of more than 128 q heads)
    const size_t pieces = (4 * (n_tokens + n_seqs) + n_seqs + 1) * sizeof(int32_t), cuts = chunk_umma_bytes(n_tokens, num_sms);
    return pieces > cuts ? pieces : cuts;
}

cudaError_t launch_chunk(const TreeArgs &args, int32_t *work, cudaStream_t st) {
    TreeArgs a = args;
    TreeParams &p = a.p;
    const bool umma = chunk_umma_fits(args), tf32_fits = p.q_type == BML_F32 && p.scale_log2 > 0.f && tree_umma_fits(a);
    const uint32_t live = args.live;
    if (umma ? p.n_seqs <= kFewSeqs && p.n_tokens <= (p.n_seqs == 1 ? kTreeMaxNodes / 2 : kFewTokens) && !p.diag
             : p.n_tokens <= kTreeMaxNodes && p.n_seqs <= kTreeMaxSeqs) {
        tree_rows(a, p.n_tokens, p.group, p.n_seqs, live, a.max_new ? a.max_new : live <= kFewSeqs ? p.n_tokens : 0u);
        return !umma && a.kv_type != BML_F32 && tf32_fits && a.rows >= kTf32Rows ? launch_tree_umma32(a, st) : launch_tree(a, st);
    }
    if (umma) return launch_chunk_umma(args, work, st);
    PieceParams pp = {};
    pp.node_start = p.node_start;
    pp.kv_lens = p.kv_lens;
    pp.n = p.n_seqs;
    pp.n_tokens = p.n_tokens;
    pp.width = p.group < kPieceRows ? kPieceRows / p.group : 1;
    pp.most = p.n_seqs + p.n_tokens / pp.width;
    pp.room = (uint64_t)p.max_pages << p.page_shift;
    pp.first = work;
    pp.start = pp.first + p.n_seqs + 1;
    pp.end = pp.start + pp.most;
    pp.lens = pp.end + pp.most;
    pp.row_of = pp.lens + pp.most;
    cudaError_t e = launch_after(chunk_pieces_kernel, dim3(1), kThreads, 0, st, pp);
    // how many pieces have tokens, and the most of one, as far as the caller said it
    tree_rows(a, p.n_tokens, p.group, pp.most, live + p.n_tokens / pp.width, a.max_new < pp.width ? a.max_new : pp.width);
    const bool tf32 = a.kv_type != BML_F32 && tf32_fits && a.rows >= kTf32Rows;
    for (uint32_t base = 0; base < pp.most && e == cudaSuccess; base += kTreeMaxSeqs) {
        p.n_seqs = pp.most - base < kTreeMaxSeqs ? pp.most - base : kTreeMaxSeqs;
        p.node_start = pp.start + base;
        p.node_end = pp.end + base;
        p.kv_lens = pp.lens + base;
        p.row_of = pp.row_of + base;
        e = tf32 ? launch_tree_umma32(a, st) : launch_tree(a, st);
    }
    return e;
}

}  // namespace bml
