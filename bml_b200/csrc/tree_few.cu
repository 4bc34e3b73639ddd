// tree_few.cu -- attention of drafted tokens over a paged cache for at most 8
// rows a kv head (plain decode among them), 16-bit pages; 16-bit queries of
// the pages' type, or 32-bit queries.
//
// The mathematics and the schedule are those of tree.cu / tree.cuh.  The work
// is to stream K and V once, so everything else is kept small: positions are
// the MMA's 16 rows and query rows its 8 columns (S^T = K Q^T, O^T = V^T P^T
// with mma.sync.m16n8k16), which halves the instructions and the registers of
// the form with 16 query rows (tree_warp.cu), and a warp's 16 positions arrive
// as one TMA box per 128-byte column block.
//
// A unit is a request with up to 8 or 16 kv heads (hpu, the largest power of
// two that divides n_kv): warp w serves head w % hpu and positions w / hpu of
// every tile, so the warps of a CTA read neighbouring 128- or 256-byte pieces
// of the same pool rows at about the same time, and a row group's heads share
// the walk over the request.  Each warp has a ring of its own and meets the
// others only at a segment's end.
//
// 32-bit queries (kQ32): terms as in tree_warp.cu.
#include <math.h>

#include "mma_frag.cuh"
#include "tree.cuh"
#include "umma.cuh"

namespace bml {

namespace {

constexpr float kGrow = 8.0f;  // log2 units a row's maximum may grow before O is rescaled
constexpr int kRows = 8;

template <int D, bool kF16, bool kQ32>
struct NCfg {
    static constexpr int TERMS = kQ32 ? (kF16 ? 2 : 3) : 1;
    static constexpr int NW = D == 128 ? 8 : 16;  // warps
    static constexpr int KB = D / 64;
    static constexpr int BOX = 16 * 128;          // bytes of a box: 16 positions x 64 values
    static constexpr int STAGE = 2 * KB * BOX;    // K then V of 16 positions
    static constexpr int NST = 3;                 // 192 KB of ring either way
    static constexpr int CH = D / 2;              // columns that meet at once
    static constexpr int CS = CH + 4;
    static constexpr int OFF_MEET = NW * NST * STAGE;
    static constexpr int OFF_ML = OFF_MEET + NW * kRows * CS * 4;
    static constexpr int OFF_BAR = OFF_ML + NW * kRows * 8;
    static constexpr int SMEM = OFF_BAR + NW * NST * 12;  // mbarriers, page flags
};

struct FewParams {
    CUtensorMap tk, tv;  // (d, n_kv, rows), box (64, 1, 16)
    TreeParams t;
    uint32_t splits;  // warps of a head
};

template <int D, bool kF16, bool kQ32>
__global__ void __launch_bounds__(NCfg<D, kF16, kQ32>::NW * 32, 1) tree_few_kernel(const __grid_constant__ FewParams fp) {
    using C = NCfg<D, kF16, kQ32>;
    constexpr int TERMS = C::TERMS, NJ = D / 16, THREADS = C::NW * 32;
    const TreeParams &p = fp.t;
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ TreeShared sh;
    __shared__ uint32_t s_abort;
    using KT = typename std::conditional<kF16, __half, __nv_bfloat16>::type;
    volatile uint32_t *abort_flag = &s_abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const uint32_t hsub = warp % p.hpu, split = warp / p.hpu;
    uint8_t *ring = smem + warp * C::NST * C::STAGE;
    float *meet = reinterpret_cast<float *>(smem + C::OFF_MEET);
    float2 *ml = reinterpret_cast<float2 *>(smem + C::OFF_ML);
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + C::OFF_BAR) + warp * C::NST;
    volatile uint32_t *flags = reinterpret_cast<volatile uint32_t *>(smem + C::OFF_BAR + C::NW * C::NST * 8) + warp * C::NST;
    const uint32_t pmask = (1u << p.page_shift) - 1;
    // K and V are read once: 131 MB in 30 us with the hint, 34 without (64 x 2000, d = 64).
    // A wider request's row groups, which read them again, lose nothing by it (20,000
    // positions, two groups, d = 128: 37.9 us, 39.8 where those take the normal policy).
    const uint64_t policy = l2_policy_evict_first();

    if (lane == 0) {
        for (int i = 0; i < C::NST; ++i) mbar_init(&full[i], 1);
        fence_mbar_init();
    }
    if (threadIdx.x == 0) {
        s_abort = 0u;
        prefetch_tmap(&fp.tk);
        prefetch_tmap(&fp.tv);
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const TreeRange range = tree_range<false>(p, &sh, blockIdx.x, gridDim.x);
    __syncthreads();  // the set-up above
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    // ------------------------------------------------------------ copies, ahead
    TreeWalk<false> fw(range);
    TreeSeg fs = {};
    uint32_t f_left = 0, f_pos = 0, f_stage = 0, f_page = 0;
    bool live = !(p.diag & kTreeStall);  // no wait has given up: after that nothing is copied any more
    const int32_t *f_table = nullptr;
    auto page_at = [&](uint32_t pos) { return pos < fs.s.L ? (uint32_t)f_table[pos >> p.page_shift] : 0xffffffffu; };
    auto fetch = [&]() {
        if (f_left == 0) {
            if (!fw.next(p, fs)) return;
            f_left = fs.t1 - fs.t0;
            f_pos = fs.t0 * p.tile + split * 16;
            f_table = tree_table(p, fs.seq);
            f_page = page_at(f_pos);
        }
        if (lane == 0 && live) {
            const bool ok = f_page < p.n_pages;
            flags[f_stage] = ok;
            if (f_pos < fs.s.L) {
                uint8_t *dst = ring + f_stage * C::STAGE;
                // a page outside the pool is read past the map's end: zeros
                const int row = (int)(ok ? (f_page << p.page_shift) + (f_pos & pmask) : p.n_pages << p.page_shift);
                mbar_arrive_expect_tx(&full[f_stage], C::STAGE);
#pragma unroll
                for (int b = 0; b < C::KB; ++b) {
                    tma_load_3d_hint(dst + b * C::BOX, &fp.tk, b * 64, (int)(fs.head + hsub), row, &full[f_stage], policy);
                    tma_load_3d_hint(dst + (C::KB + b) * C::BOX, &fp.tv, b * 64, (int)(fs.head + hsub), row, &full[f_stage], policy);
                }
            } else {
                mbar_arrive(&full[f_stage]);
            }
        }
        f_pos += p.tile;
        if (--f_left) f_page = page_at(f_pos);  // there when the next step needs it
        f_stage = f_stage + 1 == (uint32_t)C::NST ? 0 : f_stage + 1;
    };
    auto weight = [](float x) { return kQ32 ? exp2f(x) : fast_exp2(x); };
    TreeWalk<false> walk(range);
    TreeSeg sg = {};
    uint32_t stage = 0, phase = 0;
    bool first = true;
    // ldmatrix addresses inside a box: row and swizzled 16-byte column
    // K as the A operand (positions x d), V^T as the A operand (d x positions)
    const uint32_t k_row = (lane & 7) + ((lane >> 3) & 1) * 8, k_col = lane >> 4;
    const uint32_t v_row = (lane & 7) + (lane >> 4) * 8, v_col = (lane >> 3) & 1;
    while (walk.next(p, sg)) {
        const uint32_t P = sg.s.L - min(sg.s.T, sg.s.L);
        const float scale = p.scale_log2;
        float c0 = scale, c1 = scale;  // score scales of rows 2c and 2c + 1
        uint32_t q[NJ][2][TERMS];      // B operand: row g of the group, d = 16 ks + 2c (+ 8)
        {
            const bool v = (uint32_t)g < sg.rows;
            const size_t at = (v ? tree_row(p, sg, sg.row0 + g, D, hsub) : 0) + 2 * c;
            if (kQ32) {
                const float *qp = static_cast<const float *>(p.q) + at;
                float e = 1.f;
                if (kF16) {
                    float a = 0.f;
#pragma unroll
                    for (int s = 0; s < D / 8; ++s) {
                        const float2 x = v ? *reinterpret_cast<const float2 *>(qp + s * 8) : make_float2(0.f, 0.f);
                        a = fmaxf(a, fmaxf(fabsf(x.x), fabsf(x.y)));
                    }
                    a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 1));
                    a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 2));
                    const int ea = min(max((int)(__float_as_uint(a) >> 23), 11), 254);
                    e = __uint_as_float((uint32_t)(254 + 10 - ea) << 23);
                    const float back = __uint_as_float((uint32_t)(ea - 10) << 23);
                    // never 0 or infinite, as in tree_warp.cu
                    c0 = fminf(fmaxf(c0 * __shfl_sync(0xffffffffu, back, 8 * c), 1.17549435e-38f), 3.40282347e38f);
                    c1 = fminf(fmaxf(c1 * __shfl_sync(0xffffffffu, back, 8 * c + 4), 1.17549435e-38f), 3.40282347e38f);
                }
#pragma unroll
                for (int s = 0; s < NJ; ++s)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float2 x = v ? *reinterpret_cast<const float2 *>(qp + s * 16 + h * 8) : make_float2(0.f, 0.f);
                        split_pair<kF16>(x.x * e, x.y * e, q[s][h]);
                    }
            } else {
                const uint16_t *qp = static_cast<const uint16_t *>(p.q) + at;
#pragma unroll
                for (int s = 0; s < NJ; ++s)
#pragma unroll
                    for (int h = 0; h < 2; ++h) q[s][h][0] = v ? *reinterpret_cast<const uint32_t *>(qp + s * 16 + h * 8) : 0u;
            }
        }
        if (first) {  // the queries' loads are on their way with the table's
            first = false;
#pragma unroll 1
            for (int i = 0; i < C::NST - 1; ++i) fetch();
        }
        float o[NJ][4];  // O^T: d = 16 j + g (+ 8), rows 2c and 2c + 1
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;  // rows 2c, 2c + 1; l: this lane's share
        bool odd = false;  // a node has values taken as zeros

#pragma unroll 1
        for (uint32_t k = sg.t0; k < sg.t1; ++k) {
            if (!wait_bar(&full[stage], phase, abort_flag, p.wait_ns)) live = false;
            __syncwarp();  // and every lane has left the stage that fetch() fills
            fetch();
            const uint32_t base = k * p.tile + split * 16, st = stage;
            uint8_t *sk = ring + st * C::STAGE, *sv = sk + C::KB * C::BOX;
            if (++stage == (uint32_t)C::NST) {
                stage = 0;
                phase ^= 1u;
            }
            if (base >= sg.s.L || !flags[st]) continue;
            const bool edge = base + 16 > P;
            if (edge) {
                // V rows past the length become zeros, and so do nodes' values that
                // are not finite (0 * NaN is not 0); tree_nonfinite adds those to rows
                // that see them.
#pragma unroll 1
                for (int i = lane; i < 16 * C::KB * 8; i += 32) {
                    const uint32_t r = (i >> 3) & 15;
                    uint4 *v4 = reinterpret_cast<uint4 *>(sv + (i >> 7) * C::BOX + r * 128 + (i & 7) * 16);
                    if (base + r >= sg.s.L) {
                        *v4 = make_uint4(0, 0, 0, 0);
                    } else if (base + r >= P) {
                        uint16_t *v = reinterpret_cast<uint16_t *>(v4);
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (odd16<kF16>(v[e])) {
                                v[e] = 0;
                                odd = true;
                            }
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the stage's next copy
                __syncwarp();
            }
            float s[4] = {0.f, 0.f, 0.f, 0.f}, lo[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < NJ; ++ks) {
                uint32_t r[4];
                const uint32_t col = ((ks & 3) * 2 + k_col) ^ (k_row & 7);
                ldsm_x4(smem_u32(sk + (ks >> 2) * C::BOX + k_row * 128 + col * 16), r);
#pragma unroll
                for (int z = 0; z < TERMS; ++z) mma16816<kF16>(z ? lo : s, r, q[ks][0][z], q[ks][1][z]);
            }
            if (kQ32)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (fabsf(s[e]) < INFINITY) s[e] = fmaf(lo[e], 1.f / kTermScale<kF16>, s[e]);  // else an infinite K, whose lower terms are NaN
            // s[0], s[1]: position base + g, rows 2c, 2c + 1; s[2], s[3]: base + g + 8
            if (edge) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t pos = base + g + (e >> 1) * 8, row = 2 * c + (e & 1);
                    if (pos >= P && !(row < sg.rows && tree_sees(p, sg.s, (sg.row0 + row) / p.group, pos - P))) s[e] = -INFINITY;
                }
            }
            s[0] *= c0;
            s[1] *= c1;
            s[2] *= c0;
            s[3] *= c1;
            float a = fmaxf(s[0], s[2]), b = fmaxf(s[1], s[3]);
            if (__any_sync(0xffffffffu, a > m0 + kGrow || b > m1 + kGrow)) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) {
                    a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, x));
                    b = fmaxf(b, __shfl_xor_sync(0xffffffffu, b, x));
                }
                const float n0 = a > m0 + kGrow ? a : m0, n1 = b > m1 + kGrow ? b : m1;
                const float f0 = n0 == -INFINITY ? 1.f : weight(m0 - n0), f1 = n1 == -INFINITY ? 1.f : weight(m1 - n1);
                m0 = n0;
                m1 = n1;
                l0 *= f0;
                l1 *= f1;
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    o[j][0] *= f0;
                    o[j][1] *= f1;
                    o[j][2] *= f0;
                    o[j][3] *= f1;
                }
            }
            // two f16 terms: weights up to 2^15 (l and o are as much larger), away from f16's smallest step
            constexpr float up = kQ32 && kF16 ? 7.f : 0.f;
            const float u0 = (m0 == -INFINITY ? 0.f : m0) - up, u1 = (m1 == -INFINITY ? 0.f : m1) - up;
            s[0] = weight(s[0] - u0);
            s[1] = weight(s[1] - u1);
            s[2] = weight(s[2] - u0);
            s[3] = weight(s[3] - u1);
            l0 += s[0] + s[2];
            l1 += s[1] + s[3];
            // P^T as the B operand (positions x rows), rounded to the pages' type
            // (kQ32: split), one transpose of 8 x 8 each
            uint32_t pb[2][TERMS];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t t[TERMS];
                split_pair<kF16>(s[2 * h], s[2 * h + 1], t);
#pragma unroll
                for (int z = 0; z < TERMS; ++z) pb[h][z] = movm_t(t[z]);
            }
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                uint32_t r[4];
                const uint32_t col = ((j & 3) * 2 + v_col) ^ (v_row & 7);
                ldsm_x4_t(smem_u32(sv + (j >> 2) * C::BOX + v_row * 128 + col * 16), r);
                if (kQ32) {
                    float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int z = TERMS - 1; z >= 0; --z) {
                        mma16816<kF16>(x, r, pb[0][z], pb[1][z]);
                        if (kF16 && z)
#pragma unroll
                            for (int e = 0; e < 4; ++e) x[e] *= 1.f / kTermScale<kF16>;
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[j][e] += x[e];
                } else {
                    mma16816<kF16>(o[j], r, pb[0][0], pb[1][0]);
                }
            }
        }
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
            l0 += __shfl_xor_sync(0xffffffffu, l0, x);
            l1 += __shfl_xor_sync(0xffffffffu, l1, x);
        }

        // ------------------------------------------ the warps of a head meet
        // [warp][row][columns], rows of a warp's head
        odd = __any_sync(0xffffffffu, odd);
        if (g == 0) {
            ml[warp * kRows + 2 * c] = make_float2(m0, odd_sign(l0, odd));
            ml[warp * kRows + 2 * c + 1] = make_float2(m1, odd_sign(l1, odd));
        }
        const uint32_t R = kRows * p.hpu;  // a power of two that divides the thread count
        float *part = sg.slot < 2 ? tree_part(p, D, blockIdx.x, sg.slot) : nullptr;
        const uint32_t row = threadIdx.x & (R - 1), h = row / kRows, r = row % kRows;  // this thread's in what follows
        float m = -INFINITY, mu = 0.f, l = 0.f, inv = 0.f;
        bool some_odd = false;
        size_t at = 0;
#pragma unroll
        for (int ch = 0; ch < 2; ++ch) {
            float *mine = meet + warp * kRows * C::CS;
#pragma unroll
            for (int j = 0; j < NJ / 2; ++j) {
                const float *oj = o[ch * (NJ / 2) + j];
                mine[(2 * c) * C::CS + j * 16 + g] = oj[0];
                mine[(2 * c + 1) * C::CS + j * 16 + g] = oj[1];
                mine[(2 * c) * C::CS + j * 16 + g + 8] = oj[2];
                mine[(2 * c + 1) * C::CS + j * 16 + g + 8] = oj[3];
            }
            __syncthreads();
            if (r < sg.rows) {
                if (ch == 0) {
                    for (uint32_t s = 0; s < fp.splits; ++s) m = fmaxf(m, ml[(s * p.hpu + h) * kRows + r].x);
                    mu = m == -INFINITY ? 0.f : m;
                    for (uint32_t s = 0; s < fp.splits; ++s) {
                        const float2 a = ml[(s * p.hpu + h) * kRows + r];
                        l += weight(a.x - mu) * fabsf(a.y);
                        some_odd |= sign_odd(a.y);
                    }
                    if (*abort_flag) l = __int_as_float(0x7fffffff);  // a copy did not arrive: NaN
                    inv = l == 0.f ? 0.f : 1.f / l;
                    at = tree_row(p, sg, sg.row0 + r, D, h);
                    if (part && threadIdx.x < R) {
                        part[(size_t)R * D + row] = m;
                        part[(size_t)R * (D + 1) + row] = l;
                    }
                }
                for (uint32_t x4 = threadIdx.x / R; x4 < C::CH / 4; x4 += THREADS / R) {
                    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
                    for (uint32_t s = 0; s < fp.splits; ++s) {
                        const uint32_t w = (s * p.hpu + h) * kRows + r;
                        const float f = weight(ml[w].x - mu);
                        const float4 y = *reinterpret_cast<const float4 *>(meet + w * C::CS + x4 * 4);
                        acc.x += f * y.x;
                        acc.y += f * y.y;
                        acc.z += f * y.z;
                        acc.w += f * y.w;
                    }
                    const uint32_t col4 = ch * (C::CH / 4) + x4;
                    tree_nonfinite4<D, KT>(p, sg, sg.head + h, r, col4 * 4, l, some_odd, acc);
                    if (part)
                        reinterpret_cast<float4 *>(part)[col4 * R + row] = acc;
                    else if (kQ32)
                        *reinterpret_cast<float4 *>(static_cast<float *>(p.out) + at + col4 * 4) =
                            make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
                    else
                        *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p.out) + at + col4 * 4) =
                            make_uint2(pack2<kF16>(acc.x * inv, acc.y * inv), pack2<kF16>(acc.z * inv, acc.w * inv));
                }
            }
            __syncthreads();
        }
    }
    // Every copy was waited for, unless a wait gave up: then let those in
    // flight land before the shared memory goes.
    if (*abort_flag) {
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 1000000ull) {}
    }
}

bool few_map(CUtensorMap *map, const void *base, bool f16, uint32_t d, uint32_t n_kv, uint64_t rows) {
    auto enc = get_encode();
    if (!enc) return false;
    cuuint64_t dims[3] = {d, n_kv, rows};
    cuuint64_t strides[2] = {(cuuint64_t)d * 2, (cuuint64_t)d * n_kv * 2};
    cuuint32_t box[3] = {64, 1, 16};
    cuuint32_t estr[3] = {1, 1, 1};
    return enc(map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(base), dims,
               strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool kF16, bool kQ32>
cudaError_t launch_n(const TreeArgs &a, cudaStream_t st) {
    using C = NCfg<D, kF16, kQ32>;
    static_assert(C::SMEM <= 227 * 1024 - 1024, "shared memory");
    static thread_local FewParams fp;
    fp.t = a.p;
    uint32_t hpu = 1;
    while (hpu < (uint32_t)C::NW && a.p.n_kv % (2 * hpu) == 0) hpu *= 2;
    fp.splits = C::NW / hpu;
    fp.t.hpu = hpu;
    fp.t.rpg = kRows;
    fp.t.tile = 16 * fp.splits;
    fp.t.heavy_rows = 0xffffffffu;
    fp.t.heavy = fp.t.light = 1;
    // 64 requests of 200 to 4000 positions, d = 64: 25.8 us, 31 without a lead, 26.2 with
    // 8; 16 of 500 to 8000, d = 128: 45.5, 49.8, 45.7
    fp.t.lead = 6;
    if (!tree_line(fp.t)) return cudaErrorNotSupported;
    const uint64_t rows = (uint64_t)a.p.n_pages << a.p.page_shift;
    if (!few_map(&fp.tk, a.p.k, kF16, D, a.p.n_kv, rows) || !few_map(&fp.tv, a.p.v, kF16, D, a.p.n_kv, rows))
        return cudaErrorInvalidValue;
    auto kern = tree_few_kernel<D, kF16, kQ32>;
    static SmemSet set;  // one for each instantiation
    cudaError_t e = set.allow(kern, C::SMEM);
    if (e != cudaSuccess) return e;
    e = launch_after(kern, dim3(a.num_sms), C::NW * 32, C::SMEM, st, fp);
    if (e != cudaSuccess) return e;
    return launch_tree_merge(fp.t, D, a.num_sms, st);
}

template <int D>
cudaError_t launch_types(const TreeArgs &a, cudaStream_t st) {
    const bool f16 = a.kv_type == BML_F16;
    if (a.p.q_type == BML_F32) return f16 ? launch_n<D, true, true>(a, st) : launch_n<D, false, true>(a, st);
    return f16 ? launch_n<D, true, false>(a, st) : launch_n<D, false, false>(a, st);
}

}  // namespace

cudaError_t launch_tree_few(const TreeArgs &a, cudaStream_t st) {
    return a.D == 128 ? launch_types<128>(a, st) : launch_types<64>(a, st);
}

}  // namespace bml
