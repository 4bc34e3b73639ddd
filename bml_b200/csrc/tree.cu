// tree.cu -- attention of drafted tokens over a paged cache, 32-bit form,
// and the merge of divided units.
//
//   o[t,h] = sum_p softmax_p(scale * q[t,h] . k[p]) v[p]
//
// over the positions p < P = kv_len - T and the drafted nodes p = P + j that
// node t's mask names (its ancestors and itself): the attention block of
// forward_layer_cached (crates/compiler/src/gguf_compiler.rs:1008-1050 in
// SugarFreeDoNoSo/bml) for every node of a draft at once.  A row that sees
// nothing is zero.
//
// tree_f32_kernel serves 32-bit pages where tree_umma32.cu does not (the rule
// stands in launch_tree): results to about f32 precision from TF32 matrix
// instructions.  Every f32 operand is split
// x = hi + lo, hi = tf32(x), lo = tf32(x - hi) (22 bits together), and
// products are hi*hi + lo*hi + hi*lo; f16 and bf16 values are tf32 values
// already, so 16-bit pages need no lo.  A warp keeps 16 rows' output in
// registers, its positions' K and V arrive by cp.async in a private ring.
#include <math.h>

#include "tree.cuh"

namespace bml {

namespace {

constexpr int kThreads = 256;
constexpr float kGrow = 8.0f;  // log2 units a row's maximum may grow before O is rescaled
constexpr int kWarps = kThreads / 32;

__device__ __forceinline__ void mma_tf32(float *d, const uint32_t *a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float load_q(const void *q, int type, size_t i) {
    if (type == BML_F32) return static_cast<const float *>(q)[i];
    if (type == BML_F16) return __half2float(static_cast<const __half *>(q)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(q)[i]);
}
__device__ __forceinline__ void store_out4(void *out, int type, size_t i, float4 x) {
    if (type == BML_F32) {
        *reinterpret_cast<float4 *>(static_cast<float *>(out) + i) = x;
    } else if (type == BML_F16) {
        const __half2 a = __floats2half2_rn(x.x, x.y), b = __floats2half2_rn(x.z, x.w);
        *reinterpret_cast<uint2 *>(static_cast<__half *>(out) + i) =
            make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
    } else {
        const __nv_bfloat162 a = __floats2bfloat162_rn(x.x, x.y), b = __floats2bfloat162_rn(x.z, x.w);
        *reinterpret_cast<uint2 *>(static_cast<__nv_bfloat16 *>(out) + i) =
            make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
    }
}

// RW warps cover RW * 16 rows; the 8 / RW groups of RW warps take turns at
// stages of SP = 8 * RW positions.
template <int D, typename KT, int RW>
struct FCfg {
    static constexpr int ES = sizeof(KT);
    static constexpr int GROUPS = kWarps / RW;
    static constexpr int SP = 8 * RW;
    static constexpr int TILE = GROUPS * SP;  // positions of a schedule tile: a stage of every group
    // Row strides in bytes.  K: lane (g, c) reads 16-byte pieces at row g,
    // 16-byte column 2c (f32) or c (16-bit); V: at rows 2c, 2c+1, column g.
    // With these paddings the 8 lanes of a quarter-warp meet 8 bank groups.
    static constexpr int KS = D * ES + (ES == 4 ? 16 : 64);
    static constexpr int VS = D * ES + 16;
    static constexpr int STAGE = SP * (KS + VS);
    static constexpr int Q_BYTES = RW * 16 * D * 8;  // hi and lo fragments
    static constexpr int NST = 3 * GROUPS * STAGE + Q_BYTES <= 224 * 1024 ? 3 : 2;
    static constexpr int RING = GROUPS * NST * STAGE;
    static constexpr int OUT_BYTES = kWarps * 16 * (D + 4) * 4;  // combine area, over the ring
    static constexpr int MAIN = RING > OUT_BYTES ? RING : OUT_BYTES;
    static constexpr int FLAGS = GROUPS * NST * RW;  // one word per 8 positions of a stage
    static constexpr int SMEM = Q_BYTES + MAIN + FLAGS * 4;
};

template <int RW>
__device__ __forceinline__ void group_sync(int group) {
    if (RW == 1) __syncwarp();
    else named_bar_sync(1 + group, RW * 32);
}

template <int D, typename KT, int RW>
__global__ void __launch_bounds__(kThreads, 1) tree_f32_kernel(const __grid_constant__ TreeParams p) {
    using C = FCfg<D, KT, RW>;
    constexpr bool kF32 = C::ES == 4;
    constexpr int NT = D / 8;          // output column tiles of a warp
    constexpr int NB = RW;             // blocks of 8 positions at a time
    constexpr int VE = 16 / C::ES;     // V elements of one 16-byte piece
    extern __shared__ __align__(16) uint8_t smem[];
    uint32_t *sQ = reinterpret_cast<uint32_t *>(smem);
    uint8_t *ring = smem + C::Q_BYTES;
    uint32_t *flags = reinterpret_cast<uint32_t *>(ring + C::MAIN);
    __shared__ TreeShared sh;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int rw = warp % RW, grp = warp / RW, tig = rw * 32 + lane;  // thread in its group
    uint8_t *my_ring = ring + grp * C::NST * C::STAGE;
    uint32_t *my_flags = flags + grp * C::NST * RW;
    const size_t prow = (size_t)p.n_kv * D;  // elements of a pool row
    const uint32_t pmask = (1u << p.page_shift) - 1;

    asm volatile("griddepcontrol.wait;" ::: "memory");
    const TreeRange range = tree_range<false>(p, &sh, blockIdx.x, gridDim.x);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the merge, which waits for this grid
    TreeWalk<false> walk(range);
    TreeSeg sg;
    while (walk.next(p, sg)) {
        // Q fragments, split: [row warp][k-step][hi | lo][lane][4]
        for (int i = threadIdx.x; i < RW * (D / 8) * 32; i += kThreads) {
            const int l = i & 31, ks = (i >> 5) % (D / 8), w = i / (32 * (D / 8));
            const int dim = (ks >> 2) * 32 + (l & 3) * 8 + (ks & 3) * 2;
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int h8 = 0; h8 < 2; ++h8) {
                const uint32_t r = w * 16 + (l >> 2) + h8 * 8;
                float x0 = 0.f, x1 = 0.f;
                if (r < sg.rows) {
                    const size_t at = tree_row(p, sg, sg.row0 + r, D) + dim;
                    x0 = load_q(p.q, p.q_type, at);
                    x1 = load_q(p.q, p.q_type, at + 1);
                }
                tf32_split_any(x0, hi[h8], lo[h8]);
                tf32_split_any(x1, hi[h8 + 2], lo[h8 + 2]);
            }
            uint4 *dst = reinterpret_cast<uint4 *>(sQ) + ((size_t)(w * (D / 8) + ks) * 2) * 32 + l;
            dst[0] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            dst[32] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        __syncthreads();

        const uint32_t P = sg.s.L - min(sg.s.T, sg.s.L);  // committed positions
        const uint32_t pos0 = sg.t0 * C::TILE;
        const uint32_t n_steps = sg.t1 - sg.t0;
        const int32_t *table = tree_table(p, sg.seq);
        auto step_pos = [&](uint32_t k) { return pos0 + (k * C::GROUPS + grp) * C::SP; };
        // the group's copies of step k into stage k % NST
        auto fetch = [&](uint32_t k) {
            if (k < n_steps) {
                const uint32_t base = step_pos(k), st = k % C::NST;
                uint8_t *dk = my_ring + st * C::STAGE, *dv = dk + C::SP * C::KS;
                constexpr int PER = D * C::ES / 16;  // pieces of a row
#pragma unroll
                for (int i = 0; i < C::SP * PER / (RW * 32); ++i) {
                    const int piece = i * RW * 32 + tig, r = piece / PER, x = piece % PER;
                    const uint32_t pos = base + r;
                    uint32_t page = 0xffffffffu;
                    if (pos < sg.s.L) page = (uint32_t)table[pos >> p.page_shift];
                    const bool ok = page < p.n_pages;
                    const size_t at = ok ? ((((size_t)page << p.page_shift) + (pos & pmask)) * prow + (size_t)sg.head * D) * C::ES + x * 16 : 0;
                    cp16(smem_u32(dk + r * C::KS + x * 16), static_cast<const char *>(p.k) + at, ok ? 16 : 0);
                    cp16(smem_u32(dv + r * C::VS + x * 16), static_cast<const char *>(p.v) + at, ok ? 16 : 0);
                    if (x == 0 && (r & 7) == 0) my_flags[st * RW + (r >> 3)] = ok;  // 8 positions share a page
                }
            }
            cp_commit();
        };

        float o[NT][4];
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;  // rows g and g + 8; l: this lane's share
        bool odd = false;  // a node has values taken as zeros
        const uint32_t r0 = sg.row0 + rw * 16 + g, r1 = r0 + 8;
        const uint32_t t0 = r0 / p.group, t1 = r1 / p.group;
        const bool v0 = r0 < sg.row0 + sg.rows, v1 = r1 < sg.row0 + sg.rows;
        const uint4 *qf = reinterpret_cast<const uint4 *>(sQ) + (size_t)(rw * (D / 8) * 2) * 32 + lane;

#pragma unroll
        for (int i = 0; i < C::NST - 1; ++i) fetch(i);
        for (uint32_t k = 0; k < n_steps; ++k) {
            cp_wait<C::NST - 2>();
            group_sync<RW>(grp);
            fetch(k + C::NST - 1);  // into the stage that step k - 1 has left (the barrier above)
            const uint32_t st = k % C::NST;
            const uint8_t *sk = my_ring + st * C::STAGE, *sv = sk + C::SP * C::KS;
            const bool row_live = sg.rows > (uint32_t)rw * 16;
            if (!row_live) continue;
#pragma unroll 1
            for (int n0 = 0; n0 < RW; n0 += NB) {  // NB blocks of 8 positions share the Q fragments
                const uint32_t base = step_pos(k) + n0 * 8;
                uint32_t live = 0;  // bit per block: inside the length, on a page of the pool
#pragma unroll
                for (int n = 0; n < NB; ++n)
                    if (base + n * 8 < sg.s.L && my_flags[st * RW + n0 + n]) live |= 1u << n;
                if (live == 0) continue;
                // S = Q K^T: hi * hi apart from the cross terms
                float s0[NB][4], s1[NB][4];
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s0[n][e] = s1[n][e] = 0.f;
                const uint8_t *krow = sk + (n0 * 8 + g) * C::KS;
#pragma unroll
                for (int s = 0; s < D / 32; ++s) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {  // two k-steps: 16 bytes of f32, half of 16 bytes of 16-bit values
                        uint4 qh[2], ql[2];
#pragma unroll
                        for (int kk = 0; kk < 2; ++kk) {
                            qh[kk] = qf[((s * 4 + 2 * h + kk) * 2) * 32];
                            ql[kk] = qf[((s * 4 + 2 * h + kk) * 2 + 1) * 32];
                        }
#pragma unroll
                        for (int n = 0; n < NB; ++n) {
                            const uint8_t *kr = krow + n * 8 * C::KS;
                            float x[8];
                            if (kF32) Elem<float>::widen(lds128(kr + s * 128 + c * 32 + h * 16), x);
                            else Elem<KT>::widen(lds128(kr + s * 64 + c * 16), x);
                            const float *y = kF32 ? x : x + 4 * h;
#pragma unroll
                            for (int kk = 0; kk < 2; ++kk) {
                                uint32_t b0, b1, e0 = 0, e1 = 0;
                                if (kF32) {
                                    tf32_split_any(y[2 * kk], b0, e0);
                                    tf32_split_any(y[2 * kk + 1], b1, e1);
                                } else {
                                    b0 = __float_as_uint(y[2 * kk]);
                                    b1 = __float_as_uint(y[2 * kk + 1]);
                                }
                                mma_tf32(s0[n], &qh[kk].x, b0, b1);
                                mma_tf32(s1[n], &ql[kk].x, b0, b1);
                                if (kF32) mma_tf32(s1[n], &qh[kk].x, e0, e1);
                            }
                        }
                    }
                }
                const bool edge = base + NB * 8 > P;
                float a = -INFINITY, b = -INFINITY;
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    float *x = s0[n];
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = (x[e] + s1[n][e]) * p.scale_log2;
                    if (!(live >> n & 1)) x[0] = x[1] = x[2] = x[3] = -INFINITY;
                    else if (edge) {
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const uint32_t pos = base + n * 8 + 2 * c + e;
                            if (pos >= P) {
                                if (!(v0 && tree_sees(p, sg.s, t0, pos - P))) x[e] = -INFINITY;
                                if (!(v1 && tree_sees(p, sg.s, t1, pos - P))) x[2 + e] = -INFINITY;
                            }
                        }
                    }
                    a = fmaxf(a, fmaxf(x[0], x[1]));
                    b = fmaxf(b, fmaxf(x[2], x[3]));
                }
                if (__any_sync(0xffffffffu, a > m0 + kGrow || b > m1 + kGrow)) {
                    a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 1));
                    b = fmaxf(b, __shfl_xor_sync(0xffffffffu, b, 1));
                    a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 2));
                    b = fmaxf(b, __shfl_xor_sync(0xffffffffu, b, 2));
                    const float n0m = a > m0 + kGrow ? a : m0, n1m = b > m1 + kGrow ? b : m1;
                    const float f0 = n0m == -INFINITY ? 1.f : exp2f(m0 - n0m), f1 = n1m == -INFINITY ? 1.f : exp2f(m1 - n1m);
                    m0 = n0m;
                    m1 = n1m;
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
                const float u0 = m0 == -INFINITY ? 0.f : m0, u1 = m1 == -INFINITY ? 0.f : m1;
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    float *x = s0[n];
                    x[0] = exp2f(x[0] - u0);
                    x[1] = exp2f(x[1] - u0);
                    x[2] = exp2f(x[2] - u1);
                    x[3] = exp2f(x[3] - u1);
                    l0 += x[0] + x[1];
                    l1 += x[2] + x[3];
                }
                // P as the A operand: k index c is position 2c, c + 4 is 2c + 1.  The
                // matrix unit's accumulation truncates, so the NB blocks are summed
                // apart and added to O with a rounding.
                // A node's V value that is not finite is taken as zero: 0 * it must not
                // reach rows that do not see it (tree_nonfinite adds it to the others).
#pragma unroll
                for (int s = 0; s < NT / VE; ++s) {
                    float y[VE][4];
#pragma unroll
                    for (int e = 0; e < VE; ++e) y[e][0] = y[e][1] = y[e][2] = y[e][3] = 0.f;
#pragma unroll
                    for (int n = 0; n < NB; ++n) {
                        uint32_t ph[4], pl[4];
                        tf32_split(s0[n][0], ph[0], pl[0]);
                        tf32_split(s0[n][2], ph[1], pl[1]);
                        tf32_split(s0[n][1], ph[2], pl[2]);
                        tf32_split(s0[n][3], ph[3], pl[3]);
                        const uint8_t *va = sv + ((n0 + n) * 8 + 2 * c) * C::VS + g * 16, *vb = va + C::VS;
                        float y0[VE], y1[VE];
                        Elem<KT>::widen(lds128(va + s * 128), y0);
                        Elem<KT>::widen(lds128(vb + s * 128), y1);
                        if (edge) {
#pragma unroll
                            for (int e = 0; e < VE; ++e) {
                                if (!(fabsf(y0[e]) < INFINITY)) { y0[e] = 0.f; odd = true; }
                                if (!(fabsf(y1[e]) < INFINITY)) { y1[e] = 0.f; odd = true; }
                            }
                        }
#pragma unroll
                        for (int e = 0; e < VE; ++e) {
                            uint32_t b0, b1, e0 = 0, e1 = 0;
                            if (kF32) {
                                tf32_split_any(y0[e], b0, e0);
                                tf32_split_any(y1[e], b1, e1);
                            } else {
                                b0 = __float_as_uint(y0[e]);
                                b1 = __float_as_uint(y1[e]);
                            }
                            mma_tf32(y[e], pl, b0, b1);
                            if (kF32) mma_tf32(y[e], ph, e0, e1);
                            mma_tf32(y[e], ph, b0, b1);
                        }
                    }
#pragma unroll
                    for (int e = 0; e < VE; ++e)
#pragma unroll
                        for (int z = 0; z < 4; ++z) o[s * VE + e][z] += y[e][z];
                }
            }
        }
        cp_wait<0>();
        l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
        l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
        odd = __any_sync(0xffffffffu, odd);
        __syncthreads();  // the ring is free: [warp][16 rows][D + m + l], in groups' order
        constexpr int OS = D + 4;
        float *mine = reinterpret_cast<float *>(ring) + (size_t)warp * 16 * OS;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int dim = (j / VE) * 8 * VE + VE * (2 * c + e) + j % VE;
                mine[g * OS + dim] = o[j][e];
                mine[(g + 8) * OS + dim] = o[j][2 + e];
            }
        if (c == 0) {
            mine[g * OS + D] = m0;
            mine[g * OS + D + 1] = odd_sign(l0, odd);
            mine[(g + 8) * OS + D] = m1;
            mine[(g + 8) * OS + D + 1] = odd_sign(l1, odd);
        }
        __syncthreads();
        // joined over the groups: thread (row, 4 dims)
        float *part = sg.slot < 2 ? tree_part(p, D, blockIdx.x, sg.slot) : nullptr;
        for (int i = threadIdx.x; i < RW * 16 * (D / 4); i += kThreads) {
            const uint32_t r = i % (RW * 16);
            const int x4 = i / (RW * 16);
            if (r >= sg.rows) continue;
            const float *src = reinterpret_cast<float *>(ring) + ((size_t)(r / 16) * 16 + r % 16) * OS;
            constexpr size_t GS = (size_t)RW * 16 * OS;
            float m = -INFINITY;
#pragma unroll
            for (int q8 = 0; q8 < C::GROUPS; ++q8) m = fmaxf(m, src[q8 * GS + D]);
            const float mu = m == -INFINITY ? 0.f : m;
            float l = 0.f;
            bool some_odd = false;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int q8 = 0; q8 < C::GROUPS; ++q8) {
                const float f = exp2f(src[q8 * GS + D] - mu);
                const float4 y = *reinterpret_cast<const float4 *>(src + q8 * GS + x4 * 4);
                l += f * fabsf(src[q8 * GS + D + 1]);
                some_odd |= sign_odd(src[q8 * GS + D + 1]);
                // a group that saw nothing (f = 0) holds zeros
                acc.x += f * y.x;
                acc.y += f * y.y;
                acc.z += f * y.z;
                acc.w += f * y.w;
            }
            tree_nonfinite4<D, KT>(p, sg, sg.head, r, x4 * 4, l, some_odd, acc);
            if (part) {
                reinterpret_cast<float4 *>(part)[x4 * p.rpg + r] = acc;
                if (x4 == 0) {
                    part[(size_t)p.rpg * D + r] = m;
                    part[(size_t)p.rpg * (D + 1) + r] = l;
                }
            } else {
                const float inv = l == 0.f ? 0.f : 1.f / l;
                const size_t at = tree_row(p, sg, sg.row0 + r, D) + x4 * 4;
                store_out4(p.out, p.q_type, at, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
            }
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------
// Merge of the units that a cut divides.  With fewer units than cuts (by_unit)
// CTA (x, y) serves unit x, else the unit that cut x + 1 divides, if that is
// the first cut in it; it takes the unit's tasks y, y + gridDim.y, ... .
// Segments are added in a fixed order, so a result does not depend on timing.
// ---------------------------------------------------------------------------
// A joined value that came out NaN: a segment's infinity met a weight that is 0
// in 32 bits.  Such a column is the sum of the segments' values that are not
// finite.  at4: its place in a slot.
__device__ __noinline__ float4 merge_nonfinite(const TreeParams &p, uint32_t D, uint32_t first, uint32_t last, size_t at4, float4 x) {
    float o[4] = {x.x, x.y, x.z, x.w}, sum[4] = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t s = first; s <= last; ++s) {
        const float4 y = reinterpret_cast<const float4 *>(tree_part(p, D, s, s == first ? 1u : 0u))[at4];
        const float v[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (!(fabsf(v[e]) < INFINITY)) sum[e] += v[e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (sum[e] != 0.f) o[e] = sum[e];
    return make_float4(o[0], o[1], o[2], o[3]);
}

template <int D>
__global__ void __launch_bounds__(kThreads, 2) tree_merge_kernel(const __grid_constant__ TreeParams p, uint32_t grid, uint32_t by_unit) {
    __shared__ TreeShared sh;
    __shared__ float4 s_acc[2][kWarps][32];
    __shared__ float2 s_ml[kWarps][32];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    TreeSeg sg = {};
    uint32_t u0 = 0, w = 1, total = 0, b = 0;
    // (the lengths are inputs of the call, not results of the kernel before,
    // and that kernel has waited for their writer)
    bool mine;
    if (by_unit) {
        const TreeUnit u = tree_unit(p, &sh, blockIdx.x);
        mine = u.found;
        if (mine) {
            total = u.total;
            u0 = u.u0;
            w = u.w;
            sg.seq = u.seq;
            sg.head = u.head;
            sg.s = u.s;
            sg.row0 = u.rg * p.rpg;
            b = TreeCuts<true>(p, total, grid).owner(u0) + 1;  // the first cut behind u0
        }
    } else {
        b = blockIdx.x + 1;
        const TreeRange range = tree_range<true, true>(p, &sh, b, grid);
        mine = range.w0 < range.w1;
        if (mine) {
            TreeWalk<true> walk(range);
            mine = walk.next<true>(p, sg) && sg.t0 > 0;  // else the cut lies between two units
            total = range.total;
            u0 = sg.u0;
            w = sg.w;
        }
    }
    uint32_t last = 0;  // the CTAs with a segment of the unit: b - 1 to last
    if (mine) {
        const TreeCuts<true> cuts(p, total, grid);
        last = cuts.owner(u0 + (sg.s.tiles - 1) * w);
        mine = last >= b && cuts.at(b - 1) <= u0;  // divided, and no earlier cut inside the unit
        sg.rows = min(p.rpg, sg.s.rows - sg.row0);
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the segments' partials are written
    if (!mine) return;
    // A task is 8 rows x 32 columns (lane: row, twice 4 columns).  Up to 32
    // segments (8 where there is a CTA for every task): a warp a task, the loads
    // of 8 segments in flight together; more (one long request): a CTA a task,
    // the warps taking the segments in turns and meeting in shared memory.
    constexpr uint32_t kBatch = 8;
    const uint32_t R = p.rpg * p.hpu, tasks = (R + 7) / 8 * (D / 32);
    const bool many = last - b > 30 || (last - b > 6 && gridDim.y >= tasks);
    const uint32_t step = many ? kWarps : 1;
    for (uint32_t task = many ? blockIdx.y : blockIdx.y * kWarps + warp; task < tasks; task += gridDim.y * (many ? 1 : kWarps)) {
        const uint32_t row = task / (D / 32) * 8 + (lane & 7), x4 = task % (D / 32) * 8 + (lane >> 3);
        const uint32_t h = row / p.rpg, r = row - h * p.rpg;
        const bool valid = row < R && r < sg.rows;
        if (!many && !valid) continue;
        float m = -INFINITY, l = 0.f;
        float4 acc[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
        if (valid) {
            const uint32_t first = b - 1 + (many ? warp : 0);
            auto seg_part = [&](uint32_t s) { return tree_part(p, D, s, s == b - 1 ? 1u : 0u); };
            // Batches of explicit loads: a loop over segments is not unrolled so
            // that its loads overlap.  The running maximum is kept per batch.
            for (uint32_t s0 = first; s0 <= last; s0 += kBatch * step) {
                float f[kBatch], ls[kBatch];
                float4 y[kBatch][2];
#pragma unroll
                for (uint32_t u = 0; u < kBatch; ++u) {
                    const uint32_t s = s0 + u * step;
                    const float *part = seg_part(min(s, last));
                    f[u] = part[(size_t)R * D + row];
                    ls[u] = part[(size_t)R * (D + 1) + row];
                    y[u][0] = reinterpret_cast<const float4 *>(part)[x4 * R + row];
                    y[u][1] = reinterpret_cast<const float4 *>(part)[(x4 + 4) * R + row];
                }
                float mn = m;
#pragma unroll
                for (uint32_t u = 0; u < kBatch; ++u) {
                    if (s0 + u * step > last) f[u] = -INFINITY;
                    mn = fmaxf(mn, f[u]);
                }
                const float mu = mn == -INFINITY ? 0.f : mn, old = exp2f(m - mu);  // m -inf: 0
                l *= old;
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                    acc[z].x *= old;
                    acc[z].y *= old;
                    acc[z].z *= old;
                    acc[z].w *= old;
                }
#pragma unroll
                for (uint32_t u = 0; u < kBatch; ++u) {
                    if (s0 + u * step > last) continue;
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
        }
        if (many) {
            __syncthreads();
            s_acc[0][warp][lane] = acc[0];
            s_acc[1][warp][lane] = acc[1];
            s_ml[warp][lane] = make_float2(m, l);
            __syncthreads();
            if (warp != 0 || !valid) continue;
            m = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) m = fmaxf(m, s_ml[w][lane].x);
            const float mu = m == -INFINITY ? 0.f : m;
            l = 0.f;
            acc[0] = acc[1] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float2 a = s_ml[w][lane];
                const float f = exp2f(a.x - mu);
                l += f * a.y;
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                    const float4 y = s_acc[z][w][lane];
                    acc[z].x += f * y.x;
                    acc[z].y += f * y.y;
                    acc[z].z += f * y.z;
                    acc[z].w += f * y.w;
                }
            }
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const size_t at = tree_row(p, sg, sg.row0 + r, D, h) + x4 * 4;
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            const float any = (acc[z].x + acc[z].y) + (acc[z].z + acc[z].w);
            if (__builtin_expect(any != any && l == l, 0)) acc[z] = merge_nonfinite(p, D, b - 1, last, (size_t)(x4 + 4 * z) * R + row, acc[z]);
        }
#pragma unroll
        for (int z = 0; z < 2; ++z)
            store_out4(p.out, p.q_type, at + 16 * z, make_float4(acc[z].x * inv, acc[z].y * inv, acc[z].z * inv, acc[z].w * inv));
    }
}

template <int D, typename KT, int RW>
cudaError_t launch_f32(TreeParams p, int num_sms, cudaStream_t st) {
    using C = FCfg<D, KT, RW>;
    static_assert(C::SMEM <= 227 * 1024 - 512, "shared memory");
    auto kern = tree_f32_kernel<D, KT, RW>;
    static SmemSet set;  // one for each instantiation
    cudaError_t e = set.allow(kern, C::SMEM);
    if (e != cudaSuccess) return e;
    p.rpg = RW * 16;
    p.hpu = 1;
    p.tile = C::TILE;
    p.heavy_rows = 0xffffffffu;
    p.heavy = p.light = 1;
    p.lead = 2;  // 64 requests of 100 to 2000 positions, d = 64: 44.8 us, 51.7 without, 48.3 with 4
    if (!tree_line(p)) return cudaErrorNotSupported;
    e = launch_after(kern, dim3(num_sms), kThreads, C::SMEM, st, p);
    if (e != cudaSuccess) return e;
    return launch_tree_merge(p, D, num_sms, st);
}

template <int D, typename KT>
cudaError_t launch_rows(const TreeArgs &a, cudaStream_t st) {
    // Row groups of 16, whose units are more and spread better, or of 64, which read K
    // and V less often (above 16 rows this kernel is for little work, a scale of 0, and
    // groups of more than 128 q heads).
    return a.groups16() ? launch_f32<D, KT, 1>(a.p, a.num_sms, st) : launch_f32<D, KT, 4>(a.p, a.num_sms, st);
}

template <int D>
cudaError_t launch_kv(const TreeArgs &a, cudaStream_t st) {
    switch (a.kv_type) {
        case BML_F32: return launch_rows<D, float>(a, st);
        case BML_F16: return launch_rows<D, __half>(a, st);
        case BML_BF16: return launch_rows<D, __nv_bfloat16>(a, st);
    }
    return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_tree_merge(const TreeParams &p, uint32_t D, int grid, cudaStream_t st) {
    if (grid < 2) return cudaSuccess;
    const uint64_t units = tree_most_units(p);
    const bool by_unit = units < (uint64_t)(grid - 1);
    const uint32_t x = by_unit ? (uint32_t)units : (uint32_t)(grid - 1);
    // One wave of two CTAs an SM; few units (long requests) take a CTA a task.
    const uint32_t tasks = (p.rpg * p.hpu + 7) / 8 * (D / 32);
    const uint32_t most = x < 32 ? tasks : (tasks + kWarps - 1) / kWarps;
    uint32_t y = (uint32_t)grid * 2 / x;
    y = y < 1 ? 1 : y > most ? most : y;
    return D == 128 ? launch_after(tree_merge_kernel<128>, dim3(x, y), kThreads, 0, st, p, (uint32_t)grid, (uint32_t)by_unit)
                    : launch_after(tree_merge_kernel<64>, dim3(x, y), kThreads, 0, st, p, (uint32_t)grid, (uint32_t)by_unit);
}

size_t tree_workspace_bytes(uint32_t D, int num_sms) {
    return (size_t)2 * num_sms * kTreeMaxRows * (D + 2) * sizeof(float);
}

TreeForm tree_form(const TreeArgs &a) {
    // All but tree_f32_kernel scale masked scores after they were set to -inf, so a
    // scale of 0 is its.  16-bit pages: up to 8 rows a kv head (on average): the
    // form with positions as MMA rows (64 x 4000, d = 64, 8 rows: 49 us, 73 with
    // tree_warp.cu).  16-bit queries of more rows: tcgen05 where there is enough
    // work for its longer start (32 x 8000, d = 128: 24 rows 177 us against 217,
    // 64 rows 178 against 339; 12 rows 177 against 187; 64 x 4000, d = 64: 24
    // rows 82 against 93, 48 rows 78 against 144, 16 rows 82 against 74; but one
    // request of 708 positions, 4 kv heads, 64 rows 15 against 11 us).  How much
    // work there is the host knows only as a bound, the tables' width.
    // Rows count as TreeArgs::fits says: a caller that knows that most requests are
    // idle, or one much wider than the others, does not get a form that reads the
    // wide one's K and V for 8 rows at a time (1 of 131,008 positions and 64 nodes among
    // 64 places, d = 128: 170 us, 1567 with tree_few.cu).  For 32-bit queries over 16-bit
    // pages the forms differ little in a row's time and much in a request's, so the
    // average decides (60 of one token and 4 of 64, 4000 positions: 618 us in row groups
    // of 32, 917 of 64; the former one 1485 with groups of 64, 2204 with 8).
    // 32-bit pages: row groups of 16 up to 16 rows, 32 with d = 64 (64 requests of 1000
    // positions, d = 128: 16 rows 172 us, 256 on tcgen05, 20 rows 321 and 256; d = 64: 32
    // rows 94 and 103; 4 of 2000, 24 rows 18.1 and 23.1, 40 rows 23.4 and 23.6) and where
    // they make little work for its longer start: one request of 700 positions, d = 128: 20
    // rows 13.8 us, 18.2 on tcgen05, 64 rows 19.0 and 19.4, 120 rows 25.8 and 21.2; of
    // 2000: 20 rows 18.8 and 24.8, 64 rows 29.7 and 26.1; d = 64, 700: 128 rows 12.3 and
    // 14.7, 240 rows 15.6 and 15.0; 2000: 64 rows 13.2 and 13.7, 128 rows 18.3 and 15.4.
    const bool little = a.most_tiles() <= 2ull * a.num_sms;
    if (a.p.scale_log2 > 0.f && a.kv_type != BML_F32) {
        if (a.fits(8)) return TreeForm::kFew;
        const bool small = little || a.fits(a.D == 128 ? 8 : 16);
        return a.p.q_type == BML_F32 || !tree_umma_fits(a) || (small && a.fits(64)) ? TreeForm::kWarp : TreeForm::kUmma;
    }
    return a.p.scale_log2 > 0.f && tree_umma_fits(a) && !a.groups16() ? TreeForm::kUmma32 : TreeForm::kF32;
}

cudaError_t launch_tree(const TreeArgs &a, cudaStream_t st) {
    switch (tree_form(a)) {
        case TreeForm::kFew: return launch_tree_few(a, st);
        case TreeForm::kWarp: return launch_tree_warp(a, st);
        case TreeForm::kUmma: return launch_tree_umma(a, st);
        case TreeForm::kUmma32: return launch_tree_umma32(a, st);
        case TreeForm::kF32: break;
    }
    return a.D == 128 ? launch_kv<128>(a, st) : launch_kv<64>(a, st);
}

}  // namespace bml
