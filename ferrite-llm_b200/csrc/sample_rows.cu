// One token per logits row from given random numbers (fb_sample_rows): the
// rules of the reference sampler (crates/ferrite-core/src/sampling.rs:61-239)
// for many rows with settings of their own, without its host round trip.
//
// Mathematics: w_i = exp((x_i - max) / T).  In the row sorted by descending
// logit (equal logits in index order) min-p, top-p and top-k each keep a
// prefix, so the kept set is the shortest of the three and ends at one (logit,
// index) pair, the cut.  Masses are 64-bit integers in units of 2^-43 (vocab <=
// 2^19 keeps them below 2^62), summed in any order with one result; a weight
// that is not zero counts for one unit at least, so no kept token is
// unreachable.
//
// Bound: HBM for many rows (a row streams through registers once; what comes
// later reads a few of its vectors, or passes that find it in L2); a few rows
// are bound by the steps of the cluster that shares a row.  The first pass keeps
// the maximum of every group of 16-byte vectors in shared memory.  No sort of
// the row:
//  * min-p: the threshold logit is found exactly (the f32 whose binary64 weight
//    is the first to reach min_p); the survivors are the candidates;
//  * top_k <= SR_TOPK: at least top_k of the groups' maxima lie above the
//    threshold that a 256-bin count of these maxima gives, so the cut does too:
//    the logits above it are the candidates (a little over top_k of them);
//  * otherwise: counts and approximate masses of 256 bins of the distance to
//    the maximum narrow the cut down to a range of at most SR_LIST logits, all
//    above it are kept.
// One CTA ranks the candidates against each other with exact weights (no sort:
// 512 at most, a few lanes each) and draws; the cluster's other CTAs are gone by
// then.  A decision that leans on approximate masses is taken with their error
// on both sides; where that leaves it open, the exact mass of the row is summed.
// Rows whose cut falls among more than SR_LIST logits that no bin tells apart are
// bisected by key.
#include <cooperative_groups.h>
#include <math.h>

#include <type_traits>

#include "fb_internal.h"
#include "kq_common.cuh"

namespace fb {
namespace cg = cooperative_groups;

constexpr int SR_THREADS = 256;
constexpr int SR_WARPS = SR_THREADS / 32;
constexpr int SR_MAX_VOCAB = 1 << 19;
constexpr int SR_LIST = 512;    // candidates one CTA ranks
constexpr int SR_EACH = SR_LIST / SR_THREADS;
constexpr int SR_TOPK = 256;    // top_k up to here goes by the groups' maxima
constexpr int SR_BINS = 256;
constexpr int SR_CLUSTER = 16;
constexpr int SR_ROUNDS = 4;    // narrowings before the bisection
constexpr int SR_GROUPS = 48;   // groups a thread, at most
constexpr int SR_AHEAD = 4;     // vectors a thread has in flight
constexpr int SR_FLAGGED = 1024;
constexpr double SR_UNIT = 8796093022208.0;  // 2^43

using u64 = unsigned long long;

// A row's logits: rank r of the cluster has the run of `chunk` logits from r
// chunk on, its warp w the run of chunk / 8 from w chunk / 8 on, in `steps`
// steps of one 16-byte vector a lane; a group is `gsteps` of them.
struct SampleRowsArgs {
    const void *logits;
    int64_t stride;
    int vocab, chunk, steps, gsteps;
    bool vec;          // rows start on 16 bytes
    const float *temperature, *top_p, *min_p, *uniform;
    const int32_t *top_k;
    int32_t *tokens;
    float *probs;
};

template <typename T> constexpr int SR_E = 16 / (int)sizeof(T);  // logits a vector
__device__ __forceinline__ void sr_get(const uint4 &q, float (&v)[4]) {
    v[0] = __uint_as_float(q.x);
    v[1] = __uint_as_float(q.y);
    v[2] = __uint_as_float(q.z);
    v[3] = __uint_as_float(q.w);
}
template <typename T> __device__ __forceinline__ void sr_get16(const uint4 &q, float (&v)[8]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int k = 0; k < 4; k++) {
        if constexpr (std::is_same<T, __half>::value) {
            v[2 * k] = __half2float(__ushort_as_half((unsigned short)w[k]));
            v[2 * k + 1] = __half2float(__ushort_as_half((unsigned short)(w[k] >> 16)));
        } else {
            v[2 * k] = __uint_as_float(w[k] << 16);
            v[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
        }
    }
}
template <typename T> __device__ __forceinline__ void sr_unpack(const uint4 &q, float (&v)[SR_E<T>]) {
    if constexpr (sizeof(T) == 4) sr_get(q, v);
    else sr_get16<T>(q, v);
}
__device__ __forceinline__ float sr_load(const float *p, int i) { return p[i]; }
__device__ __forceinline__ float sr_load(const __half *p, int i) { return __half2float(p[i]); }
__device__ __forceinline__ float sr_load(const __nv_bfloat16 *p, int i) { return __bfloat162float(p[i]); }

// Order-preserving key of a logit (-0 as +0); 0 for NaN, which sorts below all.
__device__ __forceinline__ uint32_t sr_key(float x) {
    if (x != x) return 0u;
    const uint32_t b = __float_as_uint(__fadd_rn(x, 0.f));
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float sr_unkey(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}
// (logit, index) as one word: larger = earlier in the sorted row.
__device__ __forceinline__ u64 sr_pair(float x, int i) { return ((u64)sr_key(x) << 32) | (uint32_t)~i; }

// A row's settings.
struct RowRule {
    double scale, min_p, top_p, t;  // scale = 64 log2(e) / T; min_p 0: off; top_p 2: off
    float c;                        // log2(e) / T
    int top_k;                      // 0: off
    double u;
    bool greedy;
    __device__ __forceinline__ void load(const SampleRowsArgs &A, int64_t r) {
        const float tt = A.temperature ? A.temperature[r] : 1.f;
        const float mp = A.min_p ? A.min_p[r] : 0.f, tp = A.top_p ? A.top_p[r] : 1.f, uu = A.uniform[r];
        const int k = A.top_k ? A.top_k[r] : 0;
        greedy = tt <= 0.f;
        t = (tt != tt || greedy) ? 1.0 : (double)tt;
        scale = 92.33248261689366 / t;  // 64 log2(e) / T
        c = (float)fmin(fmax(scale * 0.015625, 1e-30), 1e30);  // (bounded: 0 c stays 0, -FLT_MAX c far below any weight)
        min_p = mp > 0.f ? fmin((double)mp, 1.0) : 0.0;
        top_p = tp < 1.f ? fmax((double)tp, 0.0) : 2.0;
        top_k = k > 0 && k < A.vocab ? k : 0;
        u = uu > 0.f ? fmin((double)uu, 1.0) : 0.0;
    }
    // exp((x - mx) / T) = 2^(z / 64), z = scale (x - mx): the table holds 2^(j / 64), and the rest |r| <= 1/2 of a
    // step is the Taylor polynomial of e^(r ln2 / 64) (argument below 0.0055: degree 4 leaves 4e-14).  Of an
    // infinite maximum only the infinite logits weigh, 1 each; NaN weighs 0.
    __device__ __forceinline__ double weight(float x, float mx, const double *table) const {
        if (mx == INFINITY) return x == mx ? 1.0 : 0.0;
        const double d = (double)x - (double)mx;
        const double z = __dmul_rn(d, scale);
        if (!(z > -68800.0)) return 0.0;  // below 2^-1075, NaN
        const double p = step(d, table, 0);
        const int e = __double2loint(__fma_rn(d, scale, 6755399441055744.0)) >> 6, e0 = e / 2;
        return __dmul_rn(__dmul_rn(p, exp64_pow2(e0)), exp64_pow2(e - e0));  // (e reaches -1075)
    }
    // 2^(z / 64 - floor) in [1, 2), or with `whole` the whole weight (z / 64 >= -900)
    __device__ __forceinline__ double step(double d, const double *table, int whole) const {
        const double q = __fma_rn(d, scale, 6755399441055744.0);  // 1.5 * 2^52: the nearest integer in the low bits
        const double r = __fma_rn(d, scale, -__dsub_rn(q, 6755399441055744.0));
        constexpr double L = 0.010830424696249145;  // ln2 / 64
        double p = __fma_rn(r, L * L * L * L / 24.0, L * L * L / 6.0);
        p = __fma_rn(p, r, L * L / 2.0);
        p = __fma_rn(p, r, L);
        p = __dmul_rn(p, r);
        const int n = __double2loint(q);
        const double t = table[n & 63];
        p = __fma_rn(t, p, t);
        return whole ? __hiloint2double(__double2hiint(p) + ((n >> 6) << 20), __double2loint(p)) : p;
    }
    static __device__ __forceinline__ u64 units(double w) {
        if (!(w > 0.0)) return 0ull;
        // w 2^43 <= 2^43: adding 2^52 leaves its nearest integer in the low mantissa bits
        const u64 n = (u64)__double_as_longlong(__fma_rn(w, SR_UNIT, 4503599627370496.0)) & 0xfffffffffffffull;
        return n ? n : 1ull;
    }
    // units(weight(x)) for a finite maximum; below `vmin` (weights under 2^-60) the long way
    __device__ __forceinline__ u64 units_of(float x, float mx, float vmin, const double *table) const {
        const double w = step((double)fmaxf(x, vmin) - (double)mx, table, 1);
        u64 n = (u64)__double_as_longlong(__fma_rn(w, SR_UNIT, 4503599627370496.0)) & 0xfffffffffffffull;
        n += n == 0;
        if (!(x >= vmin)) n = units(weight(x, mx, table));
        return n;
    }
};

template <typename V, typename Op> __device__ __forceinline__ V sr_reduce(V v, V *sh, Op op) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    V r = sh[threadIdx.x & (SR_WARPS - 1)];
#pragma unroll
    for (int o = SR_WARPS / 2; o > 0; o >>= 1) r = op(r, __shfl_xor_sync(0xffffffffu, r, o));
    return r;
}
// Exclusive sum over the block in thread order; *all gets the total.
template <typename V> __device__ __forceinline__ V sr_scan(V v, V *sh, V *all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    V incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const V y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
    }
    __syncthreads();
    if (lane == 31) sh[warp] = incl;
    __syncthreads();
    V before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < SR_WARPS; w++) {
        if (w < warp) before += sh[w];
        total += sh[w];
    }
    *all = total;
    return before + incl - v;
}

struct SrShared {
    u64 list[SR_LIST], wt[SR_LIST];            // rank 0: the candidates and their weights
    u64 seg[SR_CLUSTER * SR_WARPS];            // rank 0: kept mass of every warp's run
    u64 slot[2][SR_CLUSTER];                   // pushed by every rank
    u64 red[32];
    u64 cut, kept_mass, target;
    double table[64];
    float max_of[SR_CLUSTER], low_of[SR_CLUSTER], mass_of[SR_CLUSTER];
    float min_of[SR_CLUSTER];
    uint32_t edge[2];
    uint32_t cnt[2][SR_BINS], mass[2][SR_BINS];
    uint32_t flagged[SR_FLAGGED];              // groups to look into
    unsigned n_flagged, n_list;                // n_list, rank 0: candidates pushed
    int first_bin, last_bin, where;
    unsigned range_count, range_low;
    float m_at;
    uint32_t kmin;
};

static_assert(SR_BINS == SR_THREADS && SR_CLUSTER * SR_WARPS <= SR_THREADS, "a thread a bin, a thread a run");

template <typename T> __global__ void __launch_bounds__(SR_THREADS, 4) k_sample_rows(const SampleRowsArgs A) {
    constexpr int E = SR_E<T>;
    extern __shared__ float gmax[];  // [group][thread] largest logit
    __shared__ SrShared S;
    cg::cluster_group cl = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = cl.block_rank(), cs = cl.num_blocks();
    const int64_t row = blockIdx.x / cs;
    const T *x = static_cast<const T *>(A.logits) + row * A.stride;
    const int run = A.steps * 32 * E;                   // logits of a warp
    const int base = rank * A.chunk + warp * run;       // the warp's first
    const int ngroups = (A.steps + A.gsteps - 1) / A.gsteps;
    RowRule rule;
    rule.load(A, row);
    auto addu = [](u64 a, u64 b) { return a + b; };
    auto addf = [](float a, float b) { return a + b; };
    auto maxf = [](float a, float b) { return fmaxf(a, b); };
    auto minf = [](float a, float b) { return fminf(a, b); };

    // E logits from index i on as they are stored, NaN (never selected) behind the row
    auto fetch = [&](int i) {
        if (A.vec && i + E <= A.vocab) return __ldg(reinterpret_cast<const uint4 *>(x + i));
        uint32_t w[4] = {~0u, ~0u, ~0u, ~0u};
#pragma unroll
        for (int k = 0; k < E; k++)
            if (i + k < A.vocab) {
                if constexpr (E == 4) {
                    w[k] = __float_as_uint(x[i + k]);
                } else {
                    const uint32_t h = *reinterpret_cast<const unsigned short *>(x + i + k);
                    w[k / 2] = k & 1 ? (w[k / 2] & 0xffffu) | h << 16 : (w[k / 2] & 0xffff0000u) | h;
                }
            }
        return make_uint4(w[0], w[1], w[2], w[3]);
    };
    // f(E logits, first index) over this thread's vectors
    auto stream = [&](auto f) {
        for (int s = 0; s < A.steps; s += SR_AHEAD) {
            uint4 q[SR_AHEAD];
            const int i0 = base + (s * 32 + lane) * E;
            if (i0 - lane * E >= A.vocab) break;
#pragma unroll
            for (int k = 0; k < SR_AHEAD; k++)
                if (s + k < A.steps) q[k] = fetch(i0 + k * 32 * E);
#pragma unroll
            for (int k = 0; k < SR_AHEAD; k++)
                if (s + k < A.steps) {
                    float v[E];
                    sr_unpack<T>(q[k], v);
                    f(v, i0 + k * 32 * E);
                }
        }
    };

    // ---- the first pass: the groups' maxima, and for top-p without min-p the approximate mass (each thread's
    // relative to its own running maximum) and the lowest logit
    const bool by_topk = rule.top_k > 0 && rule.top_k <= SR_TOPK && rule.min_p == 0.0 && !rule.greedy;
    const bool has_p = rule.top_p < 1.0, cuts = rule.top_k > 0 || has_p;
    if (tid < 64) S.table[tid] = exp2((double)tid * 0.015625);
    if (tid == 0) S.n_list = S.n_flagged = 0;
    S.cnt[0][tid] = S.mass[0][tid] = 0;
    auto ex2 = [](float y) {
        float e;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(y));
        return e;
    };
    const bool online = has_p && rule.min_p == 0.0 && !rule.greedy;
    float tmax = -INFINITY, tsum = 0.f, tmin = INFINITY;
    {
        for (int g = 0; g < ngroups; g++) {
            float gm = -INFINITY;
            const int s1 = min(A.steps, (g + 1) * A.gsteps);
            for (int s = g * A.gsteps; s < s1; s += SR_AHEAD) {
                const int i0 = base + (s * 32 + lane) * E;
                if (i0 - lane * E >= A.vocab) break;
                uint4 q[SR_AHEAD];
                float m = -INFINITY;
#pragma unroll
                for (int k = 0; k < SR_AHEAD; k++)
                    q[k] = s + k < s1 ? fetch(i0 + k * 32 * E) : make_uint4(~0u, ~0u, ~0u, ~0u);
#pragma unroll
                for (int k = 0; k < SR_AHEAD; k++) {
                    float v[E];
                    sr_unpack<T>(q[k], v);
#pragma unroll
                    for (int e = 0; e < E; e++) m = fmaxf(m, v[e]);
                }
                gm = fmaxf(gm, m);
                if (online && m > -INFINITY) {
                    const float top = fmaxf(tmax, m);
                    const float off = -__fmul_rn(top, rule.c);
                    float sum = tsum > 0.f ? __fmul_rn(tsum, ex2(__fmul_rn(__fsub_rn(tmax, top), rule.c))) : 0.f;
#pragma unroll
                    for (int k = 0; k < SR_AHEAD; k++) {
                        float v[E];
                        sr_unpack<T>(q[k], v);
#pragma unroll
                        for (int e = 0; e < E; e++) {
                            // (NaN and -inf as -FLT_MAX, which weighs nothing)
                            sum += ex2(__fmaf_rn(fmaxf(v[e], -3.4028235e38f), rule.c, off));
                            tmin = fminf(tmin, v[e] > -INFINITY ? v[e] : INFINITY);
                        }
                    }
                    tsum = sum;
                    tmax = top;
                }
            }
            gmax[g * SR_THREADS + tid] = gm;
            tmax = fmaxf(tmax, gm);
        }
    }
    // f(logit, index) over the logits of the groups whose maximum satisfies pred; false: too many such groups
    auto look_into = [&](auto pred, auto f) {
        __syncthreads();
        if (tid == 0) S.n_flagged = 0;
        __syncthreads();
        for (int g = 0; g < ngroups; g++)
            if (pred(gmax[g * SR_THREADS + tid])) {
                const unsigned at = atomicAdd(&S.n_flagged, 1u);
                if (at < SR_FLAGGED) S.flagged[at] = (uint32_t)(g * SR_THREADS + tid);
            }
        __syncthreads();
        const unsigned n = S.n_flagged;
        if (n > SR_FLAGGED) return false;
        for (unsigned it = tid; it < n * A.gsteps; it += SR_THREADS) {
            const uint32_t id = S.flagged[it / A.gsteps];
            const int g = id / SR_THREADS, t = id % SR_THREADS, s = g * A.gsteps + it % A.gsteps;
            if (s >= A.steps) continue;
            const int i = rank * A.chunk + (t >> 5) * run + (s * 32 + (t & 31)) * E;
            float v[E];
            sr_unpack<T>(fetch(i), v);
#pragma unroll
            for (int k = 0; k < E; k++) f(v[k], i + k);
        }
        return true;
    };
    auto push = [&](float (SrShared::*field)[SR_CLUSTER], float v) {  // own value into every rank's [rank]
        if (tid < cs) (cl.map_shared_rank(&S, tid)->*field)[rank] = v;
    };
    const float bmax = sr_reduce(tmax, reinterpret_cast<float *>(S.red), maxf);
    const float blow = sr_reduce(tmax > -INFINITY ? tmax : INFINITY, reinterpret_cast<float *>(S.red), minf);
    float bsum = 0.f, bmin = INFINITY;
    if (online) {  // (relative to this CTA's maximum)
        bsum = sr_reduce(tsum > 0.f ? __fmul_rn(tsum, ex2(__fmul_rn(__fsub_rn(tmax, bmax), rule.c))) : 0.f,
                         reinterpret_cast<float *>(S.red), addf);
        bmin = sr_reduce(tmin, reinterpret_cast<float *>(S.red), minf);
    }
    if (cs > 1) cl.sync();  // every rank has started
    push(&SrShared::max_of, bmax);
    push(&SrShared::low_of, blow);
    push(&SrShared::mass_of, bsum);
    push(&SrShared::min_of, bmin);
    cl.sync();
    float mx = -INFINITY, low = INFINITY;  // the largest logit, the lowest of the threads' finite maxima
    for (int i = 0; i < cs; i++) {
        mx = fmaxf(mx, S.max_of[i]);
        low = fminf(low, S.low_of[i]);
    }
    const bool none = mx == -INFINITY;  // nothing finite: -inf is taken by greedy rows only, NaN by none
    if (rule.greedy || none) {
        u64 first = ~0ull;
        auto take = [&](float v, int i) {
            if (v == mx) first = min(first, (u64)i);
        };
        if (rule.greedy && !look_into([&](float m) { return m == mx; }, take))
            stream([&](float (&v)[E], int i) {
#pragma unroll
                for (int e = 0; e < E; e++) take(v[e], i + e);
            });
        first = sr_reduce(first, S.red, [](u64 a, u64 b) { return a < b ? a : b; });
        if (tid == 0) cl.map_shared_rank(&S, 0)->slot[0][rank] = first;
        cl.sync();
        if (rank == 0 && tid == 0) {
            for (int i = 0; i < cs; i++) first = min(first, S.slot[0][i]);
            A.tokens[row] = first == ~0ull ? -1 : (int)first;
            if (A.probs) A.probs[row] = first == ~0ull ? 0.f : 1.f;
        }
        return;
    }

    // ---- min-p: the lowest key whose weight reaches min_p (1: every logit but -inf and NaN)
    if (rule.min_p > 0.0) {
        if (tid < 32) {
            const float g = (float)((double)mx + rule.t * log(rule.min_p));
            uint32_t k0 = sr_key(isfinite(g) ? g : g > 0.f ? 3.4028235e38f : -3.4028235e38f);
            for (int it = 0; it < 64; it++) {  // (the guess is an ulp or two off at most)
                const uint32_t k = k0 + lane - 16;
                const float v = sr_unkey(k);
                const uint32_t ok = __ballot_sync(0xffffffffu, v <= mx && rule.weight(v, mx, S.table) >= rule.min_p) |
                                    __ballot_sync(0xffffffffu, v > mx);
                if (ok && !(ok & 1)) {
                    if (lane == 0) S.kmin = k0 + __ffs(ok) - 1 - 16;
                    break;
                }
                if (mx == INFINITY || it == 63) {
                    if (lane == 0) S.kmin = sr_key(mx);
                    break;
                }
                k0 += ok ? -31 : 31;
            }
        }
        __syncthreads();
    }
    const float xmin = rule.min_p > 0.0 ? sr_unkey(S.kmin) : -3.4028235e38f;  // survivors: x >= xmin
    const float vmin = rule.t < 1e30 ? (float)((double)mx - 41.0 * rule.t) : -3.4028235e38f;  // weight 2^-59
    auto unit_of = [&](float v) {
        return mx == INFINITY ? RowRule::units(rule.weight(v, mx, S.table)) : rule.units_of(v, mx, vmin, S.table);
    };
    // binary32 weight, relative error below 1e-5 wherever it is not negligible
    auto rough = [&](float v) {
        const float e = ex2(__fmul_rn(__fsub_rn(v, mx), rule.c));
        return v == mx ? 1.f : mx == INFINITY ? 0.f : e;
    };

    // ---- few candidates: min-p's survivors, or what lies above the groups' top_k-th largest maximum
    SrShared *lead = cl.map_shared_rank(&S, 0);
    auto to_list = [&](float v, int i) {
        const unsigned at = atomicAdd(&lead->n_list, 1u);
        if (at < SR_LIST) lead->list[at] = sr_pair(v, i);
    };
    auto too_many = [&]() {
        if (tid == 0) atomicAdd(&lead->n_list, (unsigned)SR_LIST + 1);
    };
    bool few = false;
    float m1 = 0.f;  // approximate mass of the survivors
    if (online)
        for (int i = 0; i < cs; i++)
            if (S.mass_of[i] > 0.f) m1 += __fmul_rn(S.mass_of[i], rough(S.max_of[i]));
    if (rule.min_p > 0.0) {
        few = true;
        if (!look_into([&](float m) { return m >= xmin; },
                       [&](float v, int i) {
                           if (v >= xmin) to_list(v, i);
                       }))
            too_many();
    } else if (by_topk) {
        few = true;
        const float span = __fsub_rn(mx, low);
        const float inv = span > 0.f && span < INFINITY ? __fdiv_rn((float)(SR_BINS - 1), span) : 0.f;
        // (distances beyond the threads' lowest maximum share bin 255, which cannot be the threshold)
        auto bin = [&](float v) {
            return v == mx ? 0 : (int)fminf(__fmul_rn(__fsub_rn(mx, v), inv), (float)(SR_BINS - 1));
        };
        for (int g = 0; g < ngroups; g++) {
            const float m = gmax[g * SR_THREADS + tid];
            const int b = m > -INFINITY ? bin(m) : SR_BINS - 1;
            if (b < SR_BINS - 1) atomicAdd(&S.cnt[0][b], 1u);
        }
        cl.sync();
        if (tid == 0) S.last_bin = SR_BINS;
        unsigned n = 0, all;
        for (int i = 0; i < cs; i++) n += cl.map_shared_rank(&S, i)->cnt[0][tid];
        const unsigned before = sr_scan(n, reinterpret_cast<unsigned *>(S.red), &all);
        if (before < (unsigned)rule.top_k && before + n >= (unsigned)rule.top_k) S.last_bin = tid;
        __syncthreads();
        const int last = S.last_bin;
        if (last < SR_BINS && inv > 0.f) {
            auto in = [&](float v) { return v > -INFINITY && bin(v) <= last; };
            if (!look_into(in, [&](float v, int i) {
                    if (in(v)) to_list(v, i);
                }))
                too_many();
        } else {
            few = false;  // fewer maxima than top_k, or equal ones
        }
    }

    auto value_of = [](u64 pr) { return sr_unkey((uint32_t)(pr >> 32)); };
    auto need_of = [&](double mass) { return (u64)ceil(rule.top_p * mass); };
    // The block ranks the n list entries: a group of lanes adds up, for one entry, what pred lets count.
    auto ranked = [&](int n, auto counts, auto use) {
        int g = 1;  // lanes an entry
        while (g < 32 && g * 2 * n <= SR_THREADS) g *= 2;
        for (int c = tid / g; c < (n + SR_THREADS / g - 1) / (SR_THREADS / g) * (SR_THREADS / g); c += SR_THREADS / g) {
            const u64 mine = c < n ? S.list[c] : 0;
            u64 mass = 0;
            int number = 0;
            for (int j = tid & (g - 1); j < n; j += g)
                if (counts(S.list[j], mine)) {
                    number++;
                    mass += S.wt[j];
                }
            for (int o = 1; o < g; o <<= 1) {
                number += __shfl_xor_sync(0xffffffffu, number, o);
                mass += __shfl_xor_sync(0xffffffffu, mass, o);
            }
            if (c < n && (tid & (g - 1)) == 0) use(c, mine, number, mass);
        }
    };
    // Where the cut falls in the list, with the mass and count above the list and the needed mass (its bounds lo, hi):
    // S.cut and, of the list down to it, S.kept_mass.  False where lo and hi do not agree.
    auto find_cut = [&](int n, u64 m_above, unsigned c_above, u64 lo, u64 hi) {
        if (tid == 0) S.first_bin = S.last_bin = n - 1;
        __syncthreads();
        int number_of[SR_EACH], k = 0;  // this thread's entries
        u64 mass_of[SR_EACH], pair_of[SR_EACH];
#pragma unroll
        for (int e = 0; e < SR_EACH; e++) number_of[e] = -1;
        ranked(n, [](u64 a, u64 b) { return a > b; }, [&](int c, u64 mine, int number, u64 mass) {
            const u64 run = m_above + mass + S.wt[c];
            const bool full = rule.top_k && c_above + number + 1 >= (unsigned)rule.top_k;
            if (full || (has_p && run >= lo)) atomicMin(&S.first_bin, number);
            if (full || (has_p && run >= hi)) atomicMin(&S.last_bin, number);
#pragma unroll
            for (int e = 0; e < SR_EACH; e++)
                if (e == k) {
                    number_of[e] = number;
                    mass_of[e] = mass + S.wt[c];
                    pair_of[e] = mine;
                }
            k++;
        });
        __syncthreads();
        const int at = S.first_bin;
        if (at != S.last_bin) return false;
#pragma unroll
        for (int e = 0; e < SR_EACH; e++)
            if (number_of[e] == at) {
                S.cut = pair_of[e];
                S.kept_mass = mass_of[e];
            }
        __syncthreads();
        return true;
    };

    if (few) {
        cl.sync();
        const int n = (int)min(lead->n_list, (unsigned)SR_LIST + 1);
        if (n <= SR_LIST) {
            // rank 0 goes on alone: nothing of the others is read after the barrier above, and a barrier that some
            // threads have left waits for the others only
            if (rank != 0) return;
            for (int i = tid; i < n; i += SR_THREADS) S.wt[i] = unit_of(value_of(S.list[i]));
            __syncthreads();
            u64 lo = ~0ull, hi = ~0ull;
            const bool open = has_p && rule.min_p == 0.0;  // the list does not hold all survivors
            if (open) {
                lo = need_of((double)m1 * (1.0 - 1e-4) * SR_UNIT);
                hi = need_of((double)m1 * (1.0 + 1e-4) * SR_UNIT);
            } else if (has_p) {
                u64 m = 0;
                for (int i = tid; i < n; i += SR_THREADS) m += S.wt[i];
                lo = hi = need_of((double)sr_reduce(m, S.red, addu));
            }
            if (!find_cut(n, 0, 0, lo, hi)) {
                u64 m = 0;  // the exact mass of the whole row
#pragma unroll 4
                for (int i = tid; i < A.vocab; i += SR_THREADS) {
                    const float v = sr_load(x, i);
                    const u64 w = unit_of(v);
                    if (v >= xmin) m += w;
                }
                lo = need_of((double)sr_reduce(m, S.red, addu));
                find_cut(n, 0, 0, lo, lo);
            }
            const u64 cut = S.cut, total = S.kept_mass;
            u64 target = (u64)(rule.u * (double)total);
            if (target >= total) target = total - 1;
            // mass before each kept entry in index order (the low halves hold ~index)
            ranked(n, [&](u64 a, u64 b) { return a >= cut && (uint32_t)a > (uint32_t)b; },
                   [&](int c, u64 mine, int, u64 mass) {
                       if (mine >= cut && mass <= target && target < mass + S.wt[c]) {
                           A.tokens[row] = (int)~(uint32_t)mine;
                           if (A.probs)
                               A.probs[row] = (float)(rule.weight(value_of(mine), mx, S.table) * SR_UNIT / (double)total);
                       }
                   });
            cl.sync();  // the other ranks have read n_list before they left
            return;
        }
    }

    // ---- many candidates: the cut's range by bins of the distance to the maximum
    u64 cut = 0;  // the last kept (logit, index) pair
    // survivors from xa on stay, those in xb .. xa are the range that the cut lies in
    float xa = cuts ? INFINITY : xmin, xb = xmin;
    bool to_top = cuts;  // the range still reaches the maximum
    auto side = [&](float v) { return !to_top && v >= xa ? 1 : v >= xb ? 0 : -1; };
    auto dist = [&](float v) { return v == mx ? 0.f : __fsub_rn(mx, v); };
    // kept mass of every warp's run, to rank 0
    auto push_run = [&](u64 m) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
        if (lane == 0) lead->seg[rank * SR_WARPS + warp] = m;
    };
    unsigned c_above = 0, in_range = 0;
    if (cuts) {
        // lowest survivor, and the approximate mass, as far as the first pass has not found them
        if (!online) {
            float lw = INFINITY, mass = 0.f;
            stream([&](float (&v)[E], int) {
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const bool in = v[e] >= xmin;
                    lw = in ? fminf(lw, v[e]) : lw;
                    const float p = rough(v[e]);
                    mass += in ? p : 0.f;
                }
            });
            lw = sr_reduce(lw, reinterpret_cast<float *>(S.red), minf);
            mass = sr_reduce(mass, reinterpret_cast<float *>(S.red), addf);
            cl.sync();  // the earlier values have been read
            push(&SrShared::min_of, lw);
            push(&SrShared::mass_of, mass);
            S.cnt[0][tid] = 0;
            cl.sync();
        } else if (by_topk) {
            cl.sync();  // the counts have been read
            S.cnt[0][tid] = 0;
            __syncthreads();
        }
        // a rank's approximate mass; its bins count it in units of 2^-30
        auto mass_at = [&](int i) {
            const float m = S.mass_of[i];
            return online && m > 0.f ? __fmul_rn(m, rough(S.max_of[i])) : m;
        };
        float lowest = INFINITY;
        for (int i = 0; i < cs; i++) lowest = fminf(lowest, S.min_of[i]);
        if (!online) {
            m1 = 0.f;
            for (int i = 0; i < cs; i++) m1 += S.mass_of[i];
        }
        const float step = __fmul_rn(mass_at(rank), 0x1p-30f), per = step > 0.f ? __fdiv_rn(1.f, step) : 0.f;
        // weights below 2^-43 share the last bin of the first round
        float lo = 0.f, hi = fminf(dist(lowest), __fdiv_rn(30.f, rule.c * 0.6931472f));
        float m_above = 0.f;
        for (int round = 0; round < SR_ROUNDS; round++) {
            const int buf = round & 1;
            const float width = hi - lo;
            const float inv = width > 0.f && width < INFINITY ? __fdiv_rn((float)(SR_BINS - 1), width) : 0.f;
            auto bin = [&](float v) {
                return (int)fminf(fmaxf(__fmul_rn(__fsub_rn(dist(v), lo), inv), 0.f), (float)(SR_BINS - 1));
            };
            stream([&](float (&v)[E], int) {
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const int b = bin(v[e]);
                    const uint32_t m = has_p ? __float2uint_rn(__fmul_rn(rough(v[e]), per)) : 0u;
                    if (side(v[e]) == 0) {
                        atomicAdd(&S.cnt[buf][b], 1u);
                        if (m) atomicAdd(&S.mass[buf][b], m);
                    }
                }
            });
            cl.sync();
            unsigned n = 0, n_low = 0, n_all;  // n_low: of the ranks before this one
            float m = 0.f, m_all;
            for (int i = 0; i < cs; i++) {
                const SrShared *o = cl.map_shared_rank(&S, i);
                if (i == rank) n_low = n;
                n += o->cnt[buf][tid];
                if (has_p) m += __fmul_rn((float)o->mass[buf][tid], __fmul_rn(mass_at(i), 0x1p-30f));
            }
            const unsigned nb = c_above + sr_scan(n, reinterpret_cast<unsigned *>(S.red), &n_all);
            __syncthreads();
            const float mb = m_above + sr_scan(m, reinterpret_cast<float *>(S.red), &m_all);
            // the cut is in the first bin that may complete top_k or top_p, or behind it up to the first that must
            const float need = (float)rule.top_p * m1, slack = 2e-4f * m1;
            const bool full = rule.top_k && nb + n >= (unsigned)rule.top_k;
            const bool may = n && (full || (has_p && mb + m + slack >= need));
            const bool must = n && (full || (has_p && mb + m - slack >= need));
            if (tid == 0) {
                S.first_bin = S.last_bin = SR_BINS;
                S.range_count = S.range_low = 0;
            }
            // (the buffer of the next round was read before this round's barrier)
            S.cnt[buf ^ 1][tid] = S.mass[buf ^ 1][tid] = 0;
            __syncthreads();
            if (may) atomicMin(&S.first_bin, tid);
            if (must) atomicMin(&S.last_bin, tid);
            __syncthreads();
            const int fb = S.first_bin, lb = min(S.last_bin, SR_BINS - 1);
            if (tid >= fb && tid <= lb) {
                atomicAdd(&S.range_count, n);
                atomicAdd(&S.range_low, n_low);
            }
            if (tid == fb) {
                S.m_at = mb;
                S.red[31] = nb;
            }
            // the bins' edges as keys (the lowest logit of a bin below fb, and of one up to lb): bins descend with the
            // logit, so 32 lanes close in on the first key that satisfies
            if (warp < 2) {
                const int bound = warp == 0 ? fb - 1 : lb;
                uint32_t l = sr_key(xb) - 1, h = to_top ? sr_key(mx) + 1 : sr_key(xa);  // never l, always h
                while (h - l > 1) {
                    const uint32_t k = l + (uint32_t)(((u64)(h - l) * (lane + 1)) >> 5);
                    const bool in = k >= h || (k > l && bin(sr_unkey(k)) <= bound);
                    const int w = __ffs(__ballot_sync(0xffffffffu, in)) - 1;
                    const uint32_t nh = __shfl_sync(0xffffffffu, k, w), nl = __shfl_sync(0xffffffffu, k, max(w - 1, 0));
                    h = min(nh, h);
                    l = w > 0 ? nl : l;
                }
                if (lane == 0) S.edge[warp] = h;
            }
            __syncthreads();
            if (fb >= SR_BINS) {  // nothing completes them: all survivors stay
                in_range = 0;
                xa = xb;
                to_top = false;
                break;
            }
            in_range = S.range_count;
            c_above = (unsigned)S.red[31];
            m_above = S.m_at;
            const uint32_t ka = S.edge[0], kb = S.edge[1];
            to_top = to_top && ka > sr_key(mx);
            if (!to_top) xa = sr_unkey(ka);
            xb = sr_unkey(kb);
            if (in_range <= SR_LIST) break;
            // the next round divides these bins
            const float w1 = width * (1.f / (SR_BINS - 1));
            hi = lb >= SR_BINS - 1 ? fmaxf(dist(lowest), hi) : lo + w1 * (lb + 1);
            lo = lo + w1 * fb;
        }
    }
    // ---- exact masses: above the range (kept), and of all survivors where top-p needs it; the range to rank 0
    const bool listed = in_range > 0 && in_range <= SR_LIST;
    const unsigned at0 = listed ? S.range_low : 0;  // the entries of the ranks before this one come first
    if (listed) {  // (in other cases a rank may still be reading rank 0's count)
        __syncthreads();
        if (tid == 0) S.n_list = 0;
        __syncthreads();
    }
    u64 kept = 0, m_all = 0;
    stream([&](float (&v)[E], int i) {
#pragma unroll
        for (int e = 0; e < E; e++) {
            const int s = side(v[e]);
            u64 w = 0;
            if (has_p || s > 0) w = unit_of(v[e]);
            m_all += v[e] >= xmin ? w : 0;
            kept += s > 0 ? w : 0;
            if (s == 0 && listed) lead->list[at0 + atomicAdd(&S.n_list, 1u)] = sr_pair(v[e], i + e);
        }
    });
    push_run(kept);
    m_all = sr_reduce(m_all, S.red, addu);
    if (tid == 0) lead->slot[1][rank] = m_all;
    cl.sync();
    const bool bisect = in_range > SR_LIST;
    if (bisect) {
        // over (key, index) pairs: the largest pair whose upper set completes top_k or top_p
        u64 above = 0, mass = 0;
        for (int i = 0; i < cs; i++) {
            mass += lead->slot[1][i];
            for (int j = 0; j < SR_WARPS; j++) above += lead->seg[i * SR_WARPS + j];
        }
        const u64 need = has_p ? need_of((double)mass) : ~0ull;
        u64 lo_pair = 0, hi_pair = ~0ull;
        while (hi_pair - lo_pair > 1) {
            const u64 mid = lo_pair + (hi_pair - lo_pair) / 2;
            u64 m = 0, n = 0;
            stream([&](float (&v)[E], int i) {
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (side(v[e]) == 0 && sr_pair(v[e], i + e) >= mid) {
                        n++;
                        if (has_p) m += unit_of(v[e]);
                    }
            });
            m = sr_reduce(m, S.red, addu);
            n = sr_reduce(n, S.red, addu);
            cl.sync();  // the slots of the last turn have been read
            if (tid < cs) {
                SrShared *o = cl.map_shared_rank(&S, tid);
                o->slot[0][rank] = m;
                o->slot[1][rank] = n;
            }
            cl.sync();
            m = above;
            n = c_above;
            for (int i = 0; i < cs; i++) {
                m += S.slot[0][i];
                n += S.slot[1][i];
            }
            if ((rule.top_k && n >= (u64)rule.top_k) || (has_p && m >= need && m > 0)) lo_pair = mid;
            else hi_pair = mid;
        }
        cut = lo_pair;
        stream([&](float (&v)[E], int i) {
#pragma unroll
            for (int e = 0; e < E; e++)
                if (side(v[e]) == 0 && sr_pair(v[e], i + e) >= cut) kept += unit_of(v[e]);
        });
        cl.sync();  // the runs' masses have been read
        push_run(kept);
        cl.sync();
    }
    if (rank != 0) return;
    // ---- rank 0 alone: the cut, the run that the draw falls into, the logit
    if (listed) {
        const int n = (int)in_range;
        for (int i = tid; i < n; i += SR_THREADS) S.wt[i] = unit_of(value_of(S.list[i]));
        u64 above = tid < cs * SR_WARPS ? S.seg[tid] : 0, mass = 0;
        above = sr_reduce(above, S.red, addu);
        for (int i = 0; i < cs; i++) mass += S.slot[1][i];
        const u64 need = has_p ? need_of((double)mass) : ~0ull;
        find_cut(n, above, c_above, need, need);
        cut = S.cut;
        for (int i = tid; i < n; i += SR_THREADS)
            if (S.list[i] >= cut) atomicAdd(&S.seg[(int)~(uint32_t)S.list[i] / run], S.wt[i]);
        __syncthreads();
    }
    const u64 mine = tid < cs * SR_WARPS ? S.seg[tid] : 0;
    u64 total;
    const u64 before = sr_scan(mine, S.red, &total);
    u64 target = (u64)(rule.u * (double)total);
    if (target >= total) target = total - 1;
    if (before <= target && target < before + mine) {
        S.where = tid;
        S.target = target - before;
    }
    __syncthreads();
    // the run, a piece of consecutive logits a thread
    const int piece = (run + SR_THREADS - 1) / SR_THREADS;
    const int p0 = S.where * run + tid * piece, p1 = min(min(p0 + piece, (S.where + 1) * run), A.vocab);
    auto stays = [&](float v, int i) {
        const int s = side(v);
        return s > 0 || (s == 0 && in_range > 0 && sr_pair(v, i) >= cut);
    };
    u64 sum = 0, all;
#pragma unroll 4
    for (int i = p0; i < p1; i++) {
        const float v = sr_load(x, i);
        const u64 w = unit_of(v);
        sum += stays(v, i) ? w : 0;
    }
    u64 upto = sr_scan(sum, S.red, &all);
    target = S.target;
    if (upto <= target && target < upto + sum) {
        for (int i = p0; i < p1; i++) {
            const float v = sr_load(x, i);
            if (!stays(v, i)) continue;
            const double w = rule.weight(v, mx, S.table);
            upto += RowRule::units(w);
            if (upto > target) {
                A.tokens[row] = i;
                if (A.probs) A.probs[row] = (float)(w * SR_UNIT / (double)total);
                break;
            }
        }
    }
}

// CTAs a row: as many as still find a place at once (four CTAs an SM), while
// every lane keeps at least SR_AHEAD vectors.
template <typename T> static void launch_sample_rows(fb_ctx *ctx, SampleRowsArgs A, int64_t rows) {
    constexpr int step = SR_THREADS * SR_E<T>;  // logits of one step of a CTA
    int cs = 1;
    while (cs < SR_CLUSTER && rows * cs * 2 <= 4 * ctx->num_sms && A.vocab > cs * step * SR_AHEAD) cs *= 2;
    A.steps = (A.vocab + cs * step - 1) / (cs * step);
    A.chunk = A.steps * step;
    // groups of SR_AHEAD vectors, longer ones where a thread would have more than SR_GROUPS of them
    A.gsteps = SR_AHEAD * ((A.steps + SR_AHEAD * SR_GROUPS - 1) / (SR_AHEAD * SR_GROUPS));
    const size_t smem = (size_t)((A.steps + A.gsteps - 1) / A.gsteps) * SR_THREADS * 4;
    auto kernel = k_sample_rows<T>;
    FB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    if (cs > 8) FB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)cs;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(rows * cs));
    cfg.blockDim = dim3(SR_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx->stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    FB_CUDA(cudaLaunchKernelEx(&cfg, kernel, (const SampleRowsArgs)A));
}

}  // namespace fb

using namespace fb;

extern "C" int fb_sample_rows(fb_ctx *ctx, int dtype, const void *logits_dev, int64_t row_stride, int64_t rows,
                              int vocab, const float *temperature_dev, const int32_t *top_k_dev,
                              const float *top_p_dev, const float *min_p_dev, const float *uniform_dev,
                              int32_t *tokens_dev, float *probs_dev) {
    return guarded([&] {
        FB_REQUIRE(dtype == FB_F32 || dtype == FB_F16 || dtype == FB_BF16,
                   "sample_rows: dtype must be FB_F32, FB_F16 or FB_BF16");
        FB_REQUIRE(vocab >= 1 && vocab <= SR_MAX_VOCAB, "sample_rows: vocab must be in 1..524288");
        FB_REQUIRE(rows >= 0 && rows <= 1 << 24, "sample_rows: rows must be in 0..2^24");
        FB_REQUIRE(row_stride >= 0 && (rows <= 1 || row_stride >= vocab), "sample_rows: row_stride is below vocab");
        if (rows == 0) return;
        FB_REQUIRE(ctx && logits_dev && uniform_dev && tokens_dev, "null argument");
        const size_t esz = dtype == FB_F32 ? 4 : 2;
        FB_REQUIRE(((uintptr_t)logits_dev & (esz - 1)) == 0 &&
                       (((uintptr_t)temperature_dev | (uintptr_t)top_k_dev | (uintptr_t)top_p_dev |
                         (uintptr_t)min_p_dev | (uintptr_t)uniform_dev | (uintptr_t)tokens_dev |
                         (uintptr_t)probs_dev) & 3) == 0,
                   "sample_rows: misaligned pointer");
        DeviceGuard guard(ctx->device);
        SampleRowsArgs A{};
        A.logits = logits_dev;
        A.stride = row_stride;
        A.vocab = vocab;
        A.vec = ((uintptr_t)logits_dev & 15) == 0 && (rows == 1 || row_stride % (int64_t)(16 / esz) == 0);
        A.temperature = temperature_dev;
        A.top_p = top_p_dev;
        A.min_p = min_p_dev;
        A.uniform = uniform_dev;
        A.top_k = top_k_dev;
        A.tokens = tokens_dev;
        A.probs = probs_dev;
        if (dtype == FB_F32) launch_sample_rows<float>(ctx, A, rows);
        else if (dtype == FB_F16) launch_sample_rows<__half>(ctx, A, rows);
        else launch_sample_rows<__nv_bfloat16>(ctx, A, rows);
    });
}
