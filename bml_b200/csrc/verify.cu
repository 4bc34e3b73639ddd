// verify.cu -- verification of drafted tokens: which path of a request's draft
// the target model's probabilities keep, and the token that follows it.
//
// Node 0 is the pending token and is kept.  At a kept node, with target row p and
// draft row q (the distribution that its children were drawn from, independently),
// the children are tried in node order against the residual r_k:
//   r_0 = p,  child x kept iff u < r_k(x) / q(x),  else r_(k+1) = norm(max(r_k - q, 0)).
// The residuals are never formed.  With c_0 = 0, S_0 = 1,
//   r_k = max(p - c_k q, 0) / S_k,  c_(k+1) = c_k + S_k,  S_(k+1) = sum_v max(p - c_(k+1) q, 0),
// since norm(max(r_k - q, 0)) is max(p - c_k q - S_k q, 0) up to a factor: so a
// rejection costs one pass over the two rows, and only where another child follows.
// Tokens that were picked (no draft rows): q is 1 at the token, so S loses p(x)
// and p(x) becomes 0, without a pass.
// The token behind the path is the first v with C(v) > u_next C(V - 1), C the
// prefix sums of max(p - c q, 0).  In exact arithmetic something is left of a
// residual whenever a child is rejected; of rows rounded to 16 bits p <= q may hold
// everywhere (0.996 and 1 at one token), and the token is drawn from p then.
//
// Whether a number is below another decides about tokens, so sums are f64: of
// f32 or 16-bit inputs, their order changes them by 1e-16 relatively.
//
// A cluster of 1 to 8 CTAs serves a request; each walks the tree by itself (the
// probabilities of drafted tokens are looked up at once at the start) and sums
// its part of a row; the sums meet in distributed shared memory.  What bounds it:
// latency for one request (launch, two dependent loads, a row pass: 8 picked nodes over
// 32,001 tokens 7.3 us); for a batch over a large vocabulary its passes one after
// another.  48 requests, 2 to 32 drawn nodes, 128,000 f32, 29 us, by time stamps: lookups
// 2.2, the first pass 8 (its 49 MB at 6.1 TB/s), one or two more of 5 to 7 out of L2, the
// last one 4 to 6, the search in its piece 1.0 to 1.3, then the end.  bf16 rows 36 us: f64
// sums of eight values a load do not fit 80 registers (376 bytes of spills), and the
// search takes up to 6.5.
#include <cooperative_groups.h>

#include "pages.cuh"

namespace cg = cooperative_groups;

namespace bml {

namespace {

constexpr int kThreads = 256;
constexpr uint32_t kWarps = kThreads / 32;
constexpr uint32_t kNodes = kTreeMaxNodes;
constexpr uint32_t kMostCluster = 8;
static_assert(kMostCluster * kWarps <= 64, "two pieces a lane");

struct VerifyShared {
    int32_t token[kNodes];
    float pv[kNodes], qv[kNodes], u[kNodes];
    uint32_t below[kNodes][kNodes / 32];  // children of a node, by node
    double part[2][kMostCluster];         // pass parity: the CTAs' sums
    double warp[kWarps];
    double all[kMostCluster * kWarps], all_q[kMostCluster * kWarps];  // the last pass: every warp's sum
    uint32_t out[kNodes];                 // tokens that are taken out of p
};

// A probability; what is not a positive number counts as 0.
template <typename T>
__device__ __forceinline__ float prob(T x) {
    const float f = (float)x;
    return f > 0.f && f < INFINITY ? f : 0.f;
}

// f64 of a number from 0 to below 2, by integer operations: the exponent's bias grows
// by 1023 - 127.  0 becomes 2^-127, and a subnormal f32 something below 2^-126; both
// are nothing beside a row's sum.
__device__ __forceinline__ double widen(float x) {
    const uint32_t b = __float_as_uint(x);
    return __hiloint2double((int)((b >> 3) + 0x38000000u), (int)(b << 29));
}

template <typename T>
struct alignas(16) Vec {
    static constexpr int N = 16 / sizeof(T);
    T v[N];
};

// The N values of a row from element e0 on (from a 16-byte boundary where `whole`),
// zeros outside [0, vocab), as they are stored: fewer registers than widened.
template <typename T>
__device__ __forceinline__ Vec<T> load_vec(const T *row, int64_t e0, uint32_t vocab, bool whole) {
    constexpr int N = Vec<T>::N;
    Vec<T> x;
    if (whole && e0 >= 0 && e0 + N <= (int64_t)vocab) {
        const uint4 z = __ldg(reinterpret_cast<const uint4 *>(row + e0));
        return *reinterpret_cast<const Vec<T> *>(&z);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) x.v[i] = e0 + i >= 0 && e0 + i < (int64_t)vocab ? row[e0 + i] : T(0.f);
    return x;
}
// All its bits in one word; with a bit of kOdd set, some value is negative, 2 or more,
// infinite or NaN.
template <typename T>
__device__ __forceinline__ uint32_t bits(const Vec<T> &x) {
    const uint4 z = *reinterpret_cast<const uint4 *>(&x);
    return z.x | z.y | z.z | z.w;
}
template <typename T>
constexpr uint32_t kOdd = sizeof(T) == 4 ? 0xc0000000u : 0xc000c000u;

// What a row pass sums: max(p - c q, 0), or p without some tokens.
template <typename T, bool kDraft>
struct Row {
    static constexpr int N = Vec<T>::N;
    const T *p, *q;
    uint32_t vocab;
    double c;
    const uint32_t *out;
    uint32_t n_out;
    int shift;  // elements from the row's start back to a 16-byte boundary
    bool q_ok;  // q's row lies on the same place of one
    __device__ __forceinline__ void at(const T *pr, const T *qr) {
        p = pr;
        q = qr;
        shift = (int)((reinterpret_cast<uintptr_t>(pr) & 15u) / sizeof(T));
        q_ok = kDraft && ((reinterpret_cast<uintptr_t>(pr) ^ reinterpret_cast<uintptr_t>(qr)) & 15u) == 0;
    }
    __device__ __forceinline__ uint32_t vecs() const { return (vocab + shift + N - 1) / N; }
    __device__ __forceinline__ int64_t first(uint32_t k) const { return (int64_t)k * N - shift; }
    // vector k's weights, whatever the values are
    __device__ __forceinline__ void weigh(uint32_t k, double (&w)[N]) const {
        const Vec<T> x = load_vec<T>(p, first(k), vocab, true);
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = (double)prob(x.v[i]);
        if (kDraft && c != 0.0) {
            const Vec<T> y = load_vec<T>(q, first(k), vocab, q_ok);
#pragma unroll
            for (int i = 0; i < N; ++i) w[i] = fmax(w[i] - c * (double)prob(y.v[i]), 0.0);
        }
        drop(k, w);
    }
    // zeros for the tokens that are taken out
    __device__ __forceinline__ void drop(uint32_t k, double (&w)[N]) const {
        if (!kDraft)
            for (uint32_t o = 0; o < n_out; ++o) {
                const int64_t i = (int64_t)out[o] - first(k);
#pragma unroll
                for (int j = 0; j < N; ++j)
                    if (i == j) w[j] = 0.0;
            }
    }
};

__device__ __forceinline__ double warp_sum(double t) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    return t;
}

// Sum of vectors [k0, k1) by a warp, value by value.
template <typename T, bool kDraft>
__device__ __noinline__ double slow_pass(const Row<T, kDraft> &r, uint32_t k0, uint32_t k1) {
    double s = 0.0;
    for (uint32_t k = k0 + (threadIdx.x & 31); k < k1; k += 32) {
        double w[Row<T, kDraft>::N];
        r.weigh(k, w);
#pragma unroll
        for (int i = 0; i < Row<T, kDraft>::N; ++i) s += w[i];
    }
    return warp_sum(s);
}

// Sum of vectors [k0, k1) by a warp; every lane gets it.  Instructions bound this (48
// requests, 128,000 f32: 30 an element, with every value looked at, made the call 79 us,
// these 11 make it 29): the values are probabilities, so one OR of their bits says for
// many at once that none is negative, infinite or NaN; else all is summed again value
// by value.  q is widened by integer operations beside the conversion unit, which
// takes p.
template <typename T, bool kDraft>
__device__ __forceinline__ double warp_pass(const Row<T, kDraft> &r, uint32_t k0, uint32_t k1) {
    constexpr int N = Vec<T>::N, kAtOnce = 4;
    const uint32_t lane = threadIdx.x & 31;
    double s[2] = {0.0, 0.0};
    uint32_t all = 0;
    if (kDraft && r.c != 0.0) {
        if (!r.q_ok) return slow_pass(r, k0, k1);
        for (uint32_t k = k0 + lane; k < k1; k += 32 * kAtOnce) {
            Vec<T> x[kAtOnce], y[kAtOnce];
#pragma unroll
            for (int a = 0; a < kAtOnce; ++a) {
                const bool in = k + a * 32 < k1;  // else zeros
                x[a] = load_vec<T>(r.p, r.first(k + a * 32), in ? r.vocab : 0u, true);
                y[a] = load_vec<T>(r.q, r.first(k + a * 32), in ? r.vocab : 0u, true);
            }
#pragma unroll
            for (int a = 0; a < kAtOnce; ++a) {
                all |= bits(x[a]) | bits(y[a]);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const double d = fma(-r.c, widen((float)y[a].v[i]), (double)(float)x[a].v[i]);
                    const int hi = __double2hiint(d), keep = ~(hi >> 31);  // 0 where d is negative
                    s[i & 1] += __hiloint2double(hi & keep, __double2loint(d) & keep);
                }
            }
        }
    } else {
        for (uint32_t k = k0 + lane; k < k1; k += 32 * kAtOnce) {
            Vec<T> x[kAtOnce];
#pragma unroll
            for (int a = 0; a < kAtOnce; ++a) x[a] = load_vec<T>(r.p, r.first(k + a * 32), k + a * 32 < k1 ? r.vocab : 0u, true);
#pragma unroll
            for (int a = 0; a < kAtOnce; ++a) {
                all |= bits(x[a]);
                double w[N];
#pragma unroll
                for (int i = 0; i < N; ++i) w[i] = (double)(float)x[a].v[i];
                r.drop(k + a * 32, w);
#pragma unroll
                for (int i = 0; i < N; ++i) s[i & 1] += w[i];
            }
        }
    }
    if (__any_sync(0xffffffffu, all & kOdd<T>)) return slow_pass(r, k0, k1);
    return warp_sum(s[0] + s[1]);
}

// The first element of vectors [k0, k1) whose prefix sum, from `base` on, is above
// tau; where rounding leaves none, the last element with a weight.  One warp.
template <typename T, bool kDraft>
__device__ __noinline__ int32_t warp_find(const Row<T, kDraft> &r, uint32_t k0, uint32_t k1, double base, double tau) {
    constexpr int N = Vec<T>::N;
    const uint32_t lane = threadIdx.x & 31;
    int32_t last = -1;
    for (uint32_t kb = k0; kb < k1; kb += 32) {
        const uint32_t k = kb + lane;
        double w[N];
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = 0.0;
        if (k < k1) r.weigh(k, w);
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < N; ++i) sum += w[i];
        double inc = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double a = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= (uint32_t)o) inc += a;
        }
        double at = base + (inc - sum);
        int32_t hit = -1, seen = -1;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            at += w[i];
            const int32_t e = (int32_t)(r.first(k) + i);
            if (w[i] > 0.0) {
                seen = e;
                if (hit < 0 && at > tau) hit = e;
            }
        }
        const uint32_t hits = __ballot_sync(0xffffffffu, hit >= 0), some = __ballot_sync(0xffffffffu, seen >= 0);
        if (hits) return __shfl_sync(0xffffffffu, hit, __ffs(hits) - 1);
        if (some) last = __shfl_sync(0xffffffffu, seen, 31 - __clz(some));
        base += __shfl_sync(0xffffffffu, inc, 31);
    }
    return last;
}

template <typename T, bool kDraft>
__global__ void __launch_bounds__(kThreads, 3) verify_kernel(const __grid_constant__ VerifyParams p) {
    __shared__ VerifyShared sh;
    cg::cluster_group cl = cg::this_cluster();
    const uint32_t C = cl.num_blocks(), rank = cl.block_rank(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t i = blockIdx.x / C;
    const T *target = static_cast<const T *>(p.target), *draft = static_cast<const T *>(p.draft);
    for (uint32_t k = threadIdx.x; k < kNodes * (kNodes / 32); k += kThreads) (&sh.below[0][0])[k] = 0;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int32_t a = p.node_start[i], b = p.node_start[i + 1];
    const bool ok = a >= 0 && b > a && (uint32_t)b <= p.n_tokens && b - a <= (int32_t)kNodes;
    const uint32_t T_nodes = ok ? (uint32_t)(b - a) : 0u;
    __syncthreads();
    if (threadIdx.x < T_nodes) {
        const uint32_t j = threadIdx.x;
        const int32_t up = p.parents[a + j], tok = p.tokens[a + j];
        const bool child = up >= 0 && up < (int32_t)j && (uint32_t)tok < p.vocab;
        sh.token[j] = tok;
        sh.u[j] = p.u[a + j];
        sh.pv[j] = sh.qv[j] = 0.f;
        if (child) {
            const size_t at = (size_t)(a + up) * p.vocab + tok;
            sh.pv[j] = prob(target[at]);
            if (kDraft) sh.qv[j] = prob(draft[at]);
            atomicOr(&sh.below[up][j >> 5], 1u << (j & 31));
        }
    }
    cl.sync();  // also: every CTA of the cluster runs, so its shared memory may be written

    int32_t *path = p.path + (size_t)i * p.max_path;
    const bool writes = rank == 0 && threadIdx.x == 0;
    Row<T, kDraft> row;
    row.vocab = p.vocab;
    row.c = 0.0;
    row.out = sh.out;
    row.n_out = 0;
    const uint32_t slice = C * kWarps, me = rank * kWarps + warp;
    uint32_t passes = 0, kept = 0, t = 0;
    uint32_t k0 = 0, k1 = 0;  // the warp's piece of the row
    auto piece_of = [&](uint32_t n) {  // of n vectors
        const uint32_t each = (n + slice - 1) / slice;
        k0 = min(me * each, n);
        k1 = min(k0 + each, n);
    };
    auto go = [&](uint32_t node) {
        row.at(target + (size_t)(a + node) * p.vocab, kDraft ? draft + (size_t)(a + node) * p.vocab : nullptr);
        piece_of(row.vecs());
    };
    // sum of the row over all CTAs, the same in each
    auto total = [&]() {
        const double w = warp_pass(row, k0, k1);
        if (lane == 0) sh.warp[warp] = w;
        __syncthreads();
        if (threadIdx.x < C) {
            double s = 0.0;
            for (uint32_t x = 0; x < kWarps; ++x) s += sh.warp[x];
            *cl.map_shared_rank(&sh.part[passes & 1][rank], threadIdx.x) = s;
        }
        cl.sync();
        double s = 0.0;
        for (uint32_t x = 0; x < C; ++x) s += sh.part[passes & 1][x];
        ++passes;
        return s;
    };

    if (T_nodes && p.max_path) {
        if (writes) path[0] = 0;
        kept = 1;
        while (true) {
            row.c = 0.0;
            row.n_out = 0;
            if (kept == p.max_path) break;  // its children are not looked at
            go(t);
            double mass = 1.0;
            bool known = true;  // mass is that of the residual
            uint32_t next = 0;
            for (uint32_t w = 0; w < kNodes / 32 && !next; ++w)
                for (uint32_t m = sh.below[t][w]; m; m &= m - 1) {
                    const uint32_t j = w * 32 + __ffs(m) - 1;
                    const double u = sh.u[j], pv = sh.pv[j], qv = sh.qv[j];
                    double r = pv;
                    if (kDraft) {
                        if (!known) mass = total();
                        known = true;
                        r = fmax(pv - row.c * qv, 0.0);
                    } else {
                        for (uint32_t o = 0; o < row.n_out; ++o)
                            if (sh.out[o] == (uint32_t)sh.token[j]) r = 0.0;  // has been rejected
                    }
                    if ((kDraft ? u * qv * mass : u * mass) < r) {
                        next = j;
                        break;
                    }
                    if (kDraft) {
                        row.c += mass;
                        known = false;
                    } else {
                        mass -= r;
                        __syncthreads();
                        if (threadIdx.x == 0) sh.out[row.n_out] = (uint32_t)sh.token[j];
                        __syncthreads();
                        ++row.n_out;
                    }
                }
            if (!next) break;
            t = next;
            if (writes) path[kept] = (int32_t)t;
            ++kept;
        }
    }
    if (writes) p.n_accept[i] = (int32_t)kept;
    if (rank == 0)
        for (uint32_t k = kept + threadIdx.x; k < p.max_path; k += kThreads) path[k] = -1;

    // the token behind node t, from the residual
    if (kept) {
        go(t);
        for (int again = 0; again < 2; ++again) {
            double q_sum = 0.0;
            const double w = warp_pass(row, k0, k1);
            if (kDraft && again) {  // q on its own: it may lie on another place of 16 bytes
                Row<T, kDraft> q_row = row;
                q_row.at(row.q, row.q);
                piece_of(q_row.vecs());
                q_sum = warp_pass(q_row, k0, k1);
                piece_of(row.vecs());
            }
            if (lane < C) {
                *cl.map_shared_rank(&sh.all[me], lane) = w;
                if (again) *cl.map_shared_rank(&sh.all_q[me], lane) = q_sum;
            }
            cl.sync();
            // prefix sums of the pieces, two a lane, by every warp
            const double y0 = 2 * lane < slice ? sh.all[2 * lane] : 0.0, y1 = 2 * lane + 1 < slice ? sh.all[2 * lane + 1] : 0.0;
            double inc = y0 + y1;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double v = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= (uint32_t)o) inc += v;
            }
            const double sum = __shfl_sync(0xffffffffu, inc, 31), begin = inc - (y0 + y1);
            bool drawn = sum > 0.0;
            if (kDraft && again) {
                q_sum = 0.0;
                for (uint32_t x = 0; x < slice; ++x) q_sum += sh.all_q[x];
                drawn = drawn && q_sum <= 2.0 * sum;
            }
            if (drawn) {
                // the first piece that ends above tau, or the last one with a weight
                const double tau = (double)p.u_next[i] * sum;
                const bool in0 = y0 > 0.0 && begin + y0 > tau, in1 = y1 > 0.0 && inc > tau;
                const uint32_t hits = __ballot_sync(0xffffffffu, in0 || in1), some = __ballot_sync(0xffffffffu, y0 > 0.0 || y1 > 0.0);
                const uint32_t who = hits ? __ffs(hits) - 1 : 31 - __clz(some);
                const uint32_t piece = __shfl_sync(0xffffffffu, 2 * lane + (hits ? !in0 : y1 > 0.0), who);
                const double before = __shfl_sync(0xffffffffu, hits ? (in0 ? begin : begin + y0) : (y1 > 0.0 ? begin + y0 : begin), who);
                if (piece == me) {
                    const int32_t token = warp_find(row, k0, k1, before, tau);
                    if (lane == 0) p.next[i] = token;
                }
                break;
            }
            // Nothing is left of the residual: by rounding, and the token is p's, unless q
            // sums to more than twice p (no distribution) or p itself has nothing.
            if (again && writes) p.next[i] = (int32_t)p.vocab - 1;
            cl.sync();  // sh.all has been read
            row.c = 0.0;
            row.n_out = 0;
        }
    } else if (writes) {
        p.next[i] = -1;
    }
    cl.sync();  // no CTA leaves while another writes into its shared memory
}

template <typename T>
cudaError_t verify_t(const VerifyParams &p, cudaStream_t st) {
    // as many CTAs a request as all fit the SMs at once, three on each
    uint32_t cluster = kMostCluster;
    while (cluster > 1 && (uint64_t)p.n * cluster > 3ull * p.num_sms) cluster /= 2;
    auto kern = p.draft ? verify_kernel<T, true> : verify_kernel<T, false>;
    return launch_clusters(kern, cluster, dim3(p.n * cluster), kThreads, 0, st, p);
}

}  // namespace

cudaError_t launch_verify_drafts(const VerifyParams &p, cudaStream_t st) {
    switch (p.type) {
        case BML_F32: return verify_t<float>(p, st);
        case BML_F16: return verify_t<__half>(p, st);
        case BML_BF16: return verify_t<__nv_bfloat16>(p, st);
    }
    return cudaErrorInvalidValue;
}

}  // namespace bml
