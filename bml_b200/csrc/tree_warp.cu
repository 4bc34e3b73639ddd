// tree_warp.cu -- attention of drafted tokens over a paged cache of 16-bit pages:
// 16-bit queries of the pages' type with few rows (up to 64 a kv head) or more than
// 128 q heads a kv head, and 32-bit queries of more than 8 rows, however many.
//
// The mathematics and the schedule are those of tree.cu / tree.cuh.  With few
// rows the work is to stream K and V: 4 * rows FLOP per 2-byte K/V element
// pair is far below the tensor core's rate, and what costs is latency -- of a
// call, of a segment's start and of its end.  So a warp keeps everything of
// its 16 rows in registers (Q fragments, scores, output) and works through
// its positions by itself with mma.sync.m16n8k16; a 128-row tcgen05 tile
// would spend its softmax and its epilogue on empty rows.  Its calls and the
// rule that picks it stand in tree.cu.
//
// RW warps (1, 2 or 4) cover RW * 16 rows; the 8 / RW groups of RW warps take
// turns at blocks of SP = 16 * RW positions, so that a tile of 128 positions
// is one step of every group.  A group copies its block by cp.async into its
// own ring, some steps ahead and across the ends of segments; RW == 1 needs no
// barrier at all inside a segment.  At a segment's end the groups' (m, l, o)
// meet in shared memory, 32 columns at a time.
//
// 32-bit queries (kQ32) are split into 16-bit terms of the pages' type, so
// that products are exact in the f32 sums: three bf16 terms hold all 24 bits;
// two f16 terms hold 22 of a row that is first scaled by a power of two to a
// largest value in [2^10, 2^11) (f16's range is small; split_pair).  The softmax weights
// are split the same way, and each block's P.V is summed apart and added to O
// with a rounding, since the matrix unit's own accumulation truncates.
#include <math.h>

#include "mma_frag.cuh"
#include "tree.cuh"

namespace bml {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr float kGrow = 8.0f;  // log2 units a row's maximum may grow before O is rescaled

template <int D, bool kF16, int RW, bool kQ32>
struct WCfg {
    static constexpr int TERMS = kQ32 ? (kF16 ? 2 : 3) : 1;  // 16-bit terms of a query or a weight
    static constexpr int GROUPS = kWarps / RW;
    static constexpr int SP = 16 * RW;             // positions of a group's step
    static constexpr int RS = D * 2 + 16;          // row stride: 8 rows of an ldmatrix in 8 bank groups
    static constexpr int STAGE = 2 * SP * RS;      // K then V
    // stages of a group's ring: 209 KB (139 beside the terms' 12 to 48 KB) or 184 KB
    static constexpr int NST = D == 128 ? (kQ32 ? 2 : 3) : (kQ32 ? 4 : 5);
    static constexpr int CH = 32;                  // columns that meet at once
    static constexpr int CS = CH + 4;
    static constexpr int OFF_MEET = GROUPS * NST * STAGE;
    static constexpr int OFF_ML = OFF_MEET + kWarps * 16 * CS * 4;
    static constexpr int OFF_FLAGS = OFF_ML + kWarps * 16 * 8;
    static constexpr int OFF_Q = OFF_FLAGS + GROUPS * NST * 4 * 4;  // kQ32: fragments [row warp][k-step][term][lane]
    static constexpr int SMEM = OFF_Q + (kQ32 ? RW * 16 * D * 2 * TERMS : 0);
};

template <int D, bool kF16, int RW, bool kQ32>
__global__ void __launch_bounds__(kThreads, 1) tree_warp_kernel(const __grid_constant__ TreeParams p) {
    using C = WCfg<D, kF16, RW, kQ32>;
    constexpr int TERMS = C::TERMS;
    constexpr int NT = D / 8;       // output column tiles of a warp
    constexpr int PER = D * 2 / 16; // 16-byte pieces of a row
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ TreeShared sh;
    using KT = typename std::conditional<kF16, __half, __nv_bfloat16>::type;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int rw = warp % RW, grp = warp / RW, tig = rw * 32 + lane;
    uint8_t *ring = smem + grp * C::NST * C::STAGE;
    float *meet = reinterpret_cast<float *>(smem + C::OFF_MEET);
    float2 *ml = reinterpret_cast<float2 *>(smem + C::OFF_ML);
    volatile uint32_t *flags = reinterpret_cast<volatile uint32_t *>(smem + C::OFF_FLAGS) + grp * C::NST * 4;
    const size_t prow = (size_t)p.n_kv * D * 2;  // bytes of a pool row
    const uint32_t pmask = (1u << p.page_shift) - 1;

    asm volatile("griddepcontrol.wait;" ::: "memory");
    const TreeRange range = tree_range<false>(p, &sh, blockIdx.x, gridDim.x);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    // ------------------------------------------------------------ copies, ahead
    TreeWalk<false> fw(range);
    TreeSeg fs = {};
    uint32_t f_left = 0, f_pos = 0, f_stage = 0;  // steps left of the segment, the next step's position, its stage
    auto fetch = [&]() {
        if (f_left == 0 && fw.next(p, fs)) {
            f_left = fs.t1 - fs.t0;
            f_pos = fs.t0 * kTreeTile + grp * C::SP;
        }
        if (f_left) {
            uint8_t *dk = ring + f_stage * C::STAGE, *dv = dk + C::SP * C::RS;
            const int32_t *table = tree_table(p, fs.seq);
#pragma unroll
            for (int b = 0; b < C::SP / 16; ++b) {  // 16 positions share a page
                const uint32_t pos = f_pos + b * 16;
                uint32_t page = 0xffffffffu;
                if (pos < fs.s.L) page = (uint32_t)table[pos >> p.page_shift];
                const bool ok = page < p.n_pages;
                const size_t at = ok ? (((size_t)page << p.page_shift) + (pos & pmask)) * prow + (size_t)fs.head * (D * 2) : 0;
                if (tig == 0) flags[f_stage * 4 + b] = ok;
                constexpr int ROWS = RW * 32 / PER;  // rows of one pass over the pieces
#pragma unroll
                for (int i = 0; i < 16 / ROWS; ++i) {
                    const int r = i * ROWS + tig / PER, x = (tig % PER) * 16;
                    const uint32_t n = ok && pos + r < fs.s.L ? 16u : 0u;  // rows past the length: zeros
                    const size_t src = n ? at + r * prow + x : 0;
                    cp16(smem_u32(dk + (b * 16 + r) * C::RS + x), static_cast<const char *>(p.k) + src, n);
                    cp16(smem_u32(dv + (b * 16 + r) * C::RS + x), static_cast<const char *>(p.v) + src, n);
                }
            }
            f_pos += kTreeTile;
            --f_left;
        }
        cp_commit();
        f_stage = f_stage + 1 == (uint32_t)C::NST ? 0 : f_stage + 1;
    };
    auto weight = [](float x) { return kQ32 ? exp2f(x) : fast_exp2(x); };
    auto group_sync = [&]() {
        if (RW == 1) __syncwarp();
        else named_bar_sync(1 + grp, RW * 32);
    };
#pragma unroll 1
    for (int i = 0; i < C::NST - 1; ++i) fetch();

    TreeWalk<false> walk(range);
    TreeSeg sg;
    uint32_t stage = 0;
    while (walk.next(p, sg)) {
        const uint32_t P = sg.s.L - min(sg.s.T, sg.s.L);
        const uint32_t r0 = rw * 16 + g, r1 = r0 + 8;  // this lane's rows of the group
        const bool v0 = r0 < sg.rows, v1 = r1 < sg.rows;
        const uint32_t t0 = (sg.row0 + r0) / p.group, t1 = (sg.row0 + r1) / p.group;
        uint32_t q[kQ32 ? 1 : D / 16][4];
        float c0 = p.scale_log2, c1 = p.scale_log2;  // score scales of rows g and g + 8
        uint4 *qf = reinterpret_cast<uint4 *>(smem + C::OFF_Q) + rw * (D / 16) * TERMS * 32 + lane;
        if (kQ32) {
            const float *qp = static_cast<const float *>(p.q);
            const float *q0 = qp + (v0 ? tree_row(p, sg, sg.row0 + r0, D) : 0) + 2 * c;
            const float *q1 = qp + (v1 ? tree_row(p, sg, sg.row0 + r1, D) : 0) + 2 * c;
            float e0 = 1.f, e1 = 1.f;
            if (kF16) {
                float a = 0.f, b = 0.f;
#pragma unroll 4
                for (int s = 0; s < D / 8; ++s) {
                    const float2 x = v0 ? *reinterpret_cast<const float2 *>(q0 + s * 8) : make_float2(0.f, 0.f);
                    const float2 y = v1 ? *reinterpret_cast<const float2 *>(q1 + s * 8) : make_float2(0.f, 0.f);
                    a = fmaxf(a, fmaxf(fabsf(x.x), fabsf(x.y)));
                    b = fmaxf(b, fmaxf(fabsf(y.x), fabsf(y.y)));
                }
                a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 1));
                b = fmaxf(b, __shfl_xor_sync(0xffffffffu, b, 1));
                a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 2));
                b = fmaxf(b, __shfl_xor_sync(0xffffffffu, b, 2));
                // exponents: 2^(10 - floor(log2 a)), kept where both it and its inverse are normal
                const int ea = min(max((int)(__float_as_uint(a) >> 23), 11), 254), eb = min(max((int)(__float_as_uint(b) >> 23), 11), 254);
                e0 = __uint_as_float((uint32_t)(254 + 10 - ea) << 23);
                e1 = __uint_as_float((uint32_t)(254 + 10 - eb) << 23);
                // never 0 or infinite (a masked score is -inf): scores are below 2^11 * 2^16 * D,
                // so that a scale below the smallest normal number makes all weights 1 either way
                c0 = fminf(fmaxf(c0 * __uint_as_float((uint32_t)(ea - 10) << 23), 1.17549435e-38f), 3.40282347e38f);
                c1 = fminf(fmaxf(c1 * __uint_as_float((uint32_t)(eb - 10) << 23), 1.17549435e-38f), 3.40282347e38f);
            }
#pragma unroll 2
            for (int s = 0; s < D / 16; ++s) {
                uint32_t t[4][TERMS];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float2 x = v0 ? *reinterpret_cast<const float2 *>(q0 + s * 16 + h * 8) : make_float2(0.f, 0.f);
                    const float2 y = v1 ? *reinterpret_cast<const float2 *>(q1 + s * 16 + h * 8) : make_float2(0.f, 0.f);
                    split_pair<kF16>(x.x * e0, x.y * e0, t[2 * h]);
                    split_pair<kF16>(y.x * e1, y.y * e1, t[2 * h + 1]);
                }
                if (grp == 0)
#pragma unroll
                    for (int z = 0; z < TERMS; ++z) qf[(s * TERMS + z) * 32] = make_uint4(t[0][z], t[1][z], t[2][z], t[3][z]);
            }
            __syncthreads();
        } else {
            const uint16_t *qp = static_cast<const uint16_t *>(p.q);
            const uint16_t *q0 = qp + (v0 ? tree_row(p, sg, sg.row0 + r0, D) : 0) + 2 * c;
            const uint16_t *q1 = qp + (v1 ? tree_row(p, sg, sg.row0 + r1, D) : 0) + 2 * c;
#pragma unroll
            for (int s = 0; s < (kQ32 ? 1 : D / 16); ++s) {
                q[s][0] = v0 ? *reinterpret_cast<const uint32_t *>(q0 + s * 16) : 0u;
                q[s][1] = v1 ? *reinterpret_cast<const uint32_t *>(q1 + s * 16) : 0u;
                q[s][2] = v0 ? *reinterpret_cast<const uint32_t *>(q0 + s * 16 + 8) : 0u;
                q[s][3] = v1 ? *reinterpret_cast<const uint32_t *>(q1 + s * 16 + 8) : 0u;
            }
        }
        float o[NT][4];
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;  // l: this lane's share
        bool odd = false;  // a node has values taken as zeros
        const bool live = sg.rows > (uint32_t)rw * 16;

        for (uint32_t k = sg.t0; k < sg.t1; ++k) {
            cp_wait<C::NST - 2>();
            group_sync();
            fetch();  // into the stage that every warp of the group has left
            uint8_t *sk = ring + stage * C::STAGE, *sv = sk + C::SP * C::RS;
            const uint32_t pos = k * kTreeTile + grp * C::SP;
            if (pos + C::SP > P && pos < sg.s.L) {
                // Drafted nodes' V values that are not finite become zeros here
                // (0 * NaN is not 0); tree_nonfinite adds them to rows that see them.
                bool mine = false;
                for (int i = tig; i < C::SP * PER; i += RW * 32) {
                    if (pos + i / PER < P) continue;
                    uint16_t *v = reinterpret_cast<uint16_t *>(sv + (i / PER) * C::RS + (i % PER) * 16);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (odd16<kF16>(v[e])) {
                            v[e] = 0;
                            mine = true;
                        }
                }
                if (RW == 1) {
                    odd |= __any_sync(0xffffffffu, mine);
                    __syncwarp();
                } else odd |= group_any(1 + grp, RW * 32, mine);
            }
            const uint32_t st = stage;
            stage = stage + 1 == (uint32_t)C::NST ? 0 : stage + 1;
            if (!live) continue;
#pragma unroll 1
            for (int b = 0; b < C::SP / 16; ++b) {
                const uint32_t base = pos + b * 16;
                if (base >= sg.s.L || !flags[st * 4 + b]) continue;
                float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
                float lo[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};  // kQ32: the smaller terms' sums
                const uint8_t *ka = sk + (b * 16 + (lane & 7) + ((lane >> 4) << 3)) * C::RS + ((lane >> 3) & 1) * 16;
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks) {
                    uint32_t r[4];
                    ldsm_x4(smem_u32(ka + ks * 32), r);
                    if (kQ32) {
#pragma unroll
                        for (int z = 0; z < TERMS; ++z) {
                            const uint4 x = qf[(ks * TERMS + z) * 32];
                            const uint32_t a4[4] = {x.x, x.y, x.z, x.w};
                            mma16816<kF16>(z ? lo[0] : s[0], a4, r[0], r[1]);
                            mma16816<kF16>(z ? lo[1] : s[1], a4, r[2], r[3]);
                        }
                    } else {
                        mma16816<kF16>(s[0], q[kQ32 ? 0 : ks], r[0], r[1]);
                        mma16816<kF16>(s[1], q[kQ32 ? 0 : ks], r[2], r[3]);
                    }
                }
                if (kQ32)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (fabsf(s[h][e]) < INFINITY) s[h][e] = fmaf(lo[h][e], 1.f / kTermScale<kF16>, s[h][e]);  // else an infinite K, whose lower terms are NaN
                if (base + 16 > P) {
                    const uint32_t w0 = v0 ? tree_see16(p, sg.s, t0, (int32_t)(base - P)) : 0u;
                    const uint32_t w1 = v1 ? tree_see16(p, sg.s, t1, (int32_t)(base - P)) : 0u;
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            if (!(w0 >> (h * 8 + 2 * c + e) & 1)) s[h][e] = -INFINITY;
                            if (!(w1 >> (h * 8 + 2 * c + e) & 1)) s[h][2 + e] = -INFINITY;
                        }
                }
                float a = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
                float d = fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3]));
                a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 1));
                d = fmaxf(d, __shfl_xor_sync(0xffffffffu, d, 1));
                a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 2));
                d = fmaxf(d, __shfl_xor_sync(0xffffffffu, d, 2));
                a *= c0;  // > 0
                d *= c1;
                if (__any_sync(0xffffffffu, a > m0 + kGrow || d > m1 + kGrow)) {
                    const float n0 = a > m0 + kGrow ? a : m0, n1 = d > m1 + kGrow ? d : m1;
                    const float f0 = n0 == -INFINITY ? 1.f : weight(m0 - n0), f1 = n1 == -INFINITY ? 1.f : weight(m1 - n1);
                    m0 = n0;
                    m1 = n1;
                    l0 *= f0;
                    l1 *= f1;
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        o[j][0] *= f0;
                        o[j][1] *= f0;
                        o[j][2] *= f1;
                        o[j][3] *= f1;
                    }
                }
                // two f16 terms: weights up to 2^15 (l and o are as much larger), away from f16's smallest step
                constexpr float up = kQ32 && kF16 ? 7.f : 0.f;
                const float u0 = (m0 == -INFINITY ? 0.f : m0) - up, u1 = (m1 == -INFINITY ? 0.f : m1) - up;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        s[h][e] = weight(fmaf(s[h][e], c0, -u0));
                        s[h][2 + e] = weight(fmaf(s[h][2 + e], c1, -u1));
                    }
                l0 += (s[0][0] + s[0][1]) + (s[1][0] + s[1][1]);
                l1 += (s[0][2] + s[0][3]) + (s[1][2] + s[1][3]);
                // P as the A operand of P.V, rounded to the pages' type (kQ32: split)
                uint32_t pa[TERMS][4];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        uint32_t t[TERMS];
                        split_pair<kF16>(s[h][2 * e], s[h][2 * e + 1], t);
#pragma unroll
                        for (int z = 0; z < TERMS; ++z) pa[z][2 * h + e] = t[z];
                    }
                const uint8_t *va = sv + (b * 16 + (lane & 7) + ((lane >> 3) & 1) * 8) * C::RS + (lane >> 4) * 16;
#pragma unroll
                for (int j = 0; j < NT; j += 2) {
                    uint32_t r[4];
                    ldsm_x4_t(smem_u32(va + j * 16), r);
                    if (kQ32) {
                        float x[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
                        for (int z = TERMS - 1; z >= 0; --z) {
                            mma16816<kF16>(x[0], pa[z], r[0], r[1]);
                            mma16816<kF16>(x[1], pa[z], r[2], r[3]);
                            if (kF16 && z)
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    x[0][e] *= 1.f / kTermScale<kF16>;
                                    x[1][e] *= 1.f / kTermScale<kF16>;
                                }
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            o[j][e] += x[0][e];
                            o[j + 1][e] += x[1][e];
                        }
                    } else {
                        mma16816<kF16>(o[j], pa[0], r[0], r[1]);
                        mma16816<kF16>(o[j + 1], pa[0], r[2], r[3]);
                    }
                }
            }
        }
        l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
        l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 2);

        // ---------------------------------------------------- the groups meet
        if (c == 0) {
            ml[warp * 16 + g] = make_float2(m0, odd_sign(l0, odd));
            ml[warp * 16 + g + 8] = make_float2(m1, odd_sign(l1, odd));
        }
        float *part = sg.slot < 2 ? tree_part(p, D, blockIdx.x, sg.slot) : nullptr;
#pragma unroll
        for (int ch = 0; ch < D / C::CH; ++ch) {
            float *mine = meet + warp * 16 * C::CS;
#pragma unroll
            for (int j = 0; j < C::CH / 8; ++j) {
                const float *oj = o[ch * (C::CH / 8) + j];
                *reinterpret_cast<float2 *>(mine + g * C::CS + j * 8 + 2 * c) = make_float2(oj[0], oj[1]);
                *reinterpret_cast<float2 *>(mine + (g + 8) * C::CS + j * 8 + 2 * c) = make_float2(oj[2], oj[3]);
            }
            __syncthreads();
            for (int i = threadIdx.x; i < RW * 16 * (C::CH / 4); i += kThreads) {
                const uint32_t r = i % (RW * 16), x4 = i / (RW * 16);
                if (r >= sg.rows) continue;
                float m = -INFINITY;
#pragma unroll
                for (int q8 = 0; q8 < C::GROUPS; ++q8) m = fmaxf(m, ml[q8 * RW * 16 + r].x);
                const float mu = m == -INFINITY ? 0.f : m;
                float l = 0.f;
                bool some_odd = false;
                float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int q8 = 0; q8 < C::GROUPS; ++q8) {
                    const float2 a = ml[q8 * RW * 16 + r];
                    const float f = weight(a.x - mu);
                    const float4 y = *reinterpret_cast<const float4 *>(meet + (q8 * RW * 16 + r) * C::CS + x4 * 4);
                    l += f * fabsf(a.y);
                    some_odd |= sign_odd(a.y);
                    acc.x += f * y.x;
                    acc.y += f * y.y;
                    acc.z += f * y.z;
                    acc.w += f * y.w;
                }
                const uint32_t col4 = ch * (C::CH / 4) + x4;
                tree_nonfinite4<D, KT>(p, sg, sg.head, r, col4 * 4, l, some_odd, acc);
                if (part) {
                    reinterpret_cast<float4 *>(part)[col4 * p.rpg + r] = acc;
                    if (col4 == 0) {
                        part[(size_t)p.rpg * D + r] = m;
                        part[(size_t)p.rpg * (D + 1) + r] = l;
                    }
                } else {
                    const float inv = l == 0.f ? 0.f : 1.f / l;
                    const size_t at = tree_row(p, sg, sg.row0 + r, D) + col4 * 4;
                    if (kQ32)
                        *reinterpret_cast<float4 *>(static_cast<float *>(p.out) + at) =
                            make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
                    else
                        *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p.out) + at) =
                            make_uint2(pack2<kF16>(acc.x * inv, acc.y * inv), pack2<kF16>(acc.z * inv, acc.w * inv));
                }
            }
            __syncthreads();
        }
    }
    cp_wait<0>();
}

template <int D, bool kF16, int RW, bool kQ32>
cudaError_t launch_w(TreeParams p, int num_sms, cudaStream_t st) {
    using C = WCfg<D, kF16, RW, kQ32>;
    static_assert(C::SMEM <= 227 * 1024 - 512, "shared memory");
    auto kern = tree_warp_kernel<D, kF16, RW, kQ32>;
    static SmemSet set;  // one for each instantiation
    cudaError_t e = set.allow(kern, C::SMEM);
    if (e != cudaSuccess) return e;
    p.rpg = RW * 16;
    p.hpu = 1;
    p.tile = kTreeTile;
    p.heavy_rows = 0xffffffffu;
    p.heavy = p.light = 1;
    p.lead = 1;  // 64 requests of 100 to 2000 positions, d = 64, 32-bit queries: 59.8 us, 70.6 without, 61.4 with 3
    if (!tree_line(p)) return cudaErrorNotSupported;
    e = launch_after(kern, dim3(num_sms), kThreads, C::SMEM, st, p);
    if (e != cudaSuccess) return e;
    return launch_tree_merge(p, D, num_sms, st);
}

template <int D, bool kF16, bool kQ32>
cudaError_t launch_rows(const TreeArgs &a, cudaStream_t st) {
    if (a.fits(16)) return launch_w<D, kF16, 1, kQ32>(a.p, a.num_sms, st);
    if (a.fits(32)) return launch_w<D, kF16, 2, kQ32>(a.p, a.num_sms, st);
    return launch_w<D, kF16, 4, kQ32>(a.p, a.num_sms, st);
}

template <int D>
cudaError_t launch_types(const TreeArgs &a, cudaStream_t st) {
    const bool f16 = a.kv_type == BML_F16;
    if (a.p.q_type == BML_F32) return f16 ? launch_rows<D, true, true>(a, st) : launch_rows<D, false, true>(a, st);
    return f16 ? launch_rows<D, true, false>(a, st) : launch_rows<D, false, false>(a, st);
}

}  // namespace

cudaError_t launch_tree_warp(const TreeArgs &a, cudaStream_t st) {
    return a.D == 128 ? launch_types<128>(a, st) : launch_types<64>(a, st);
}

}  // namespace bml
