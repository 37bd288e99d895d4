// One token per logits row from given random numbers (fb_sample_rows): the
// rules of the reference sampler (crates/ferrite-core/src/sampling.rs:61-239)
// for many rows with settings of their own, without its host round trip and its
// repetition penalty.
//
// Mathematics: w_i = exp((x_i - max) / T).  In the row sorted by descending
// logit (equal logits in index order) min-p, top-p and top-k each keep a
// prefix, so the kept set is the shortest of the three and ends at one (logit,
// index) pair, the cut.  Masses are 64-bit integers in units of 2^-43 (vocab <=
// 2^19 keeps them below 2^62), summed in any order with one result; a weight
// counts for its whole units and one more (none where exp is 0), so no kept token
// is unreachable.
//
// Bound: many rows by the first pass, which streams a row through registers once
// (an exponential a logit where top-p asks: 53 % of the issue slots and 37 % of the
// special-function unit at 31 % of DRAM's rate; what comes later reads a few of a
// row's vectors, or passes that find it in L2); a few rows by the steps of the
// cluster that shares a row.  The first pass keeps
// the maximum of every group of 16-byte vectors in shared memory.  Measured
// (back to back in a graph): 400 rows of 151936 bf16 logits, top-k 50 and top-p,
// in 45 us (48 us from cold caches, 2.5 TB/s: a row is one CTA and three of them
// share an SM); 65 rows of 128256 f32 logits, top-p alone, in 75 us, some 16 us each
// for counting into bins and for the exact masses; one row of 151936 in 8.7 us.  No
// sort of the row:
//  * min-p: the threshold logit is found exactly (the f32 whose binary64 weight
//    is the first to reach min_p); the survivors are the candidates;
//  * top_k <= SR_TOPK: at least top_k of the groups' maxima lie above the
//    threshold that a 512-bin count of these maxima gives, so the cut does too:
//    the logits above it are the candidates (a little over top_k of them);
//  * otherwise: counts and approximate masses of 512 bins of the distance to
//    the maximum narrow the cut down to a range of at most SR_LIST logits, all
//    above it are kept.
// One CTA orders the candidates (ranked against each other up to 256, else by a
// bitonic sort), adds up their exact weights and draws; the cluster's other CTAs are gone by
// then.  A decision that leans on approximate masses is taken with their error
// on both sides; where that leaves it open, the exact mass of the row is summed.
// Where no bins come down to SR_LIST logits (top-k alone far below the maximum in
// temperatures, top-p so near 1 that the masses' error spans more, many equal
// logits, temperatures that leave f32 no approximate mass: above 10^36, or beyond
// 10^30 and 10^-30 with logits near its size) bins of (key, index) pairs with exact
// masses close in on the cut, 9 bits a pass.  (65 rows of 151936: top-k 1000 at T
// 0.1 120 us, top-p 0.999 at T 0.7 184 us.)
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
constexpr int SR_RANKED = 256;  // up to here every candidate is compared with all others (182: 2 us less than sorted)
constexpr int SR_TOPK = 256;    // top_k up to here goes by the groups' maxima
constexpr int SR_BINS = 512;
constexpr int SR_CLUSTER = 16;
constexpr int SR_ROUNDS = 3;    // narrowings by distance (two are enough unless the masses' error spans more than the list)
constexpr int SR_GROUPS = 48;   // groups a thread, at most
constexpr int SR_AHEAD = 4;     // vectors a thread has in flight
constexpr int SR_FLAGGED = 1024;
constexpr float SR_REF = 4194304.f;  // 2^22: below it f32 has integers and halves
constexpr double SR_UNIT = 8796093022208.0;  // 2^43

using u64 = unsigned long long;
constexpr u64 SR_BIAS = 0x4330000000000000ull - 1;  // the bits of 2^52, less each weight's extra unit

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
// Larger logit of each place (the other one where one is NaN).
__device__ __forceinline__ uint32_t sr_max32(uint32_t a, uint32_t b, float) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
}
__device__ __forceinline__ uint32_t sr_max32(uint32_t a, uint32_t b, __half) {
    const __half2 m = __hmax2(*reinterpret_cast<__half2 *>(&a), *reinterpret_cast<__half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&m);
}
__device__ __forceinline__ uint32_t sr_max32(uint32_t a, uint32_t b, __nv_bfloat16) {
    const __nv_bfloat162 m = __hmax2(*reinterpret_cast<__nv_bfloat162 *>(&a), *reinterpret_cast<__nv_bfloat162 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&m);
}
template <typename T> __device__ __forceinline__ uint4 sr_max(const uint4 &a, const uint4 &b) {
    return make_uint4(sr_max32(a.x, b.x, T{}), sr_max32(a.y, b.y, T{}), sr_max32(a.z, b.z, T{}),
                      sr_max32(a.w, b.w, T{}));
}
// The lowest finite f32 or bf16 in every place.
template <typename T> __device__ __forceinline__ uint4 sr_lowest() {
    const uint32_t w = sizeof(T) == 4 ? 0xff7fffffu : 0xff7fff7fu;
    return make_uint4(w, w, w, w);
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
    double scale, min_p, top_p, t;  // scale = 16 log2(e) / T; min_p 0: off; top_p 2: off
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
        scale = 23.083120654223414 / t;  // 16 log2(e) / T
        c = (float)fmin(fmax(scale * 0.0625, 1e-30), 1e30);  // (bounded: 0 c stays 0, -FLT_MAX c far below any weight)
        min_p = mp > 0.f ? fmin((double)mp, 1.0) : 0.0;
        top_p = tp < 1.f ? fmax((double)tp, 0.0) : 2.0;
        top_k = k > 0 && k < A.vocab ? k : 0;
        u = uu > 0.f ? fmin((double)uu, 1.0) : 0.0;
    }
    // exp((x - mx) / T) = 2^(z / 16), z = scale (x - mx): the table holds 2^(j / 16), and the rest |r| <= 1/2 of a
    // step is the Taylor polynomial of e^(r ln2 / 16) (argument below 0.022: degree 6 leaves 5e-16).  Sixteen doubles
    // are one line of shared memory, which 32 lanes look up without a conflict; the polynomial's shorter form with 64
    // of them took longer.  Of an infinite maximum only the infinite logits weigh, 1 each; NaN weighs 0.
    __device__ __forceinline__ double weight(float x, float mx, const double *table) const {
        if (mx == INFINITY) return x == mx ? 1.0 : 0.0;
        const double d = (double)x - (double)mx;
        const double z = __dmul_rn(d, scale);
        if (!(z > -17200.0)) return 0.0;  // below 2^-1075, NaN
        const double p = step(d, table, 0);
        const int e = __double2loint(__fma_rn(d, scale, 6755399441055744.0)) >> 4, e0 = e / 2;
        return __dmul_rn(__dmul_rn(p, exp64_pow2(e0)), exp64_pow2(e - e0));  // (e reaches -1075)
    }
    // 2^(z / 16 - floor) in [1, 2), or with `whole` the whole weight (z / 16 >= -900)
    __device__ __forceinline__ double step(double d, const double *table, int whole) const {
        const double q = __fma_rn(d, scale, 6755399441055744.0);  // 1.5 * 2^52: the nearest integer in the low bits
        const double r = __fma_rn(d, scale, -__dsub_rn(q, 6755399441055744.0));
        constexpr double L = 0.04332169878499658;  // ln2 / 16
        double p = __fma_rn(r, L * L * L * L * L * L / 720.0, L * L * L * L * L / 120.0);
        p = __fma_rn(p, r, L * L * L * L / 24.0);
        p = __fma_rn(p, r, L * L * L / 6.0);
        p = __fma_rn(p, r, L * L / 2.0);
        p = __fma_rn(p, r, L);
        p = __dmul_rn(p, r);
        const int n = __double2loint(q);
        const double t = table[n & 15];
        p = __fma_rn(t, p, t);
        return whole ? __hiloint2double(__double2hiint(p) + ((n >> 4) << 20), __double2loint(p)) : p;
    }
    // One unit and the whole units of the weight, as a double (exact: at most 2^43 + 1), for a finite maximum and x >=
    // the lowest logit that weighs at all.  vmin is the lowest f32 from max - 41 T on (weights of 2^-59): what lies below
    // it weighs one unit, and the next f32 above it may be the maximum itself.
    __device__ __forceinline__ double units_of(float x, float mx, float vmin, const double *table) const {
        const double w = step((double)fmaxf(x, vmin) - (double)mx, table, 1);
        const double u = __dsub_rn(__fma_rd(w, SR_UNIT, 4503599627370496.0), 4503599627370495.0);  // + 2^52 - (2^52 - 1)
        return x < vmin ? 1.0 : u;
    }
    // The same as an integer that is SR_BIAS too large: what adds up many of them adds integers and takes the surplus
    // off once.  mx is finite here, and x above it counts as it.
    __device__ __forceinline__ u64 biased_units(float x, float mx, float vmin, const double *table) const {
        const double w = step((double)fminf(fmaxf(x, vmin), mx) - (double)mx, table, 1);
        const u64 u = (u64)__double_as_longlong(__fma_rd(w, SR_UNIT, 4503599627370496.0));
        return x < vmin ? SR_BIAS + 1 : u;
    }
    // f mass, exactly, of an f32 f in 0 .. 1 (M 2^-e, M below 2^24, e from 23 on) and a mass below 2^62: rounded down,
    // rest whether anything was dropped.
    static __device__ __forceinline__ u64 share(double f, u64 mass, bool &rest) {
        rest = false;
        if (!(f > 0.0)) return 0;
        const long long bits = __double_as_longlong(f);
        const u64 M = (u64)((bits & 0xfffffffffffffll) | 0x10000000000000ll) >> 29;
        const int e = 1023 + 23 - (int)(bits >> 52);
        const u64 hi = __umul64hi(mass, M), lo = mass * M;
        rest = e >= 64 || lo << (64 - e) != 0;  // (from 64 on: taken so, below one token's mass either way)
        return e < 64 ? hi << (64 - e) | lo >> e : e < 128 ? hi >> (e - 64) : 0;
    }
    // The mass that top-p asks for, rounded up, and the place of u in a mass: exact, so that equal weights share a
    // border as they should.
    __device__ __forceinline__ u64 need(u64 mass) const {
        bool rest;
        const u64 n = share(top_p, mass, rest);
        return n + rest;
    }
    __device__ __forceinline__ u64 place(u64 mass) const {
        bool rest;
        return min(share(u, mass, rest), mass - 1);
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
    double table[16];
    float max_of[SR_CLUSTER], low_of[SR_CLUSTER];
    double mass_of[SR_CLUSTER];
    uint32_t edge[2];
    alignas(8) uint32_t cnt[2][SR_BINS], mass[2][SR_BINS];
    uint32_t flagged[SR_FLAGGED];              // groups to look into
    unsigned n_flagged, n_list;                // n_list, rank 0: candidates pushed
    int first_bin, last_bin, where;
    unsigned range_count, range_low;
    float m_at;
    uint32_t kmin;
};

static_assert(SR_AHEAD == 4 && SR_BINS == 2 * SR_THREADS && SR_CLUSTER * SR_WARPS <= SR_THREADS,
              "a sum of four, a thread two bins, a thread a run");

template <typename T> __global__ void __launch_bounds__(SR_THREADS, 3) k_sample_rows(const SampleRowsArgs A) {
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
    auto csync = [&]() {
        if (cs > 1) cl.sync();
        else __syncthreads();
    };
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

    // ---- the first pass: the groups' maxima, and for top-p without min-p the approximate mass.  Each thread's is
    // relative to 2^ref of its own running maximum, ref an integer (within SR_REF): x c - ref is one rounding, and a
    // change of ref exact.  What it is off by: 2^-22 a term (ex2), 2^-24 |x c - ref| of it and half as much for c
    // (together 1e-6: |x c - ref| is below 17 on average over a row's mass), 10 2^-24 for a batch's sum; from there on
    // it is a double.  2.3e-6 with the last factors.
    const bool by_topk = rule.top_k > 0 && rule.top_k <= SR_TOPK && rule.min_p == 0.0 && !rule.greedy;
    const bool has_p = rule.top_p < 1.0, cuts = rule.top_k > 0 || has_p;
    if (tid < 16) S.table[tid] = exp2((double)tid * 0.0625);
    if (tid == 0) S.n_list = S.n_flagged = 0;
    for (int i = tid; i < SR_BINS; i += SR_THREADS) S.cnt[0][i] = S.mass[0][i] = 0;
    auto ex2 = [](float y) {
        float e;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(y));
        return e;
    };
    auto ref = [&](float top) { return fminf(fmaxf(ceilf(__fmul_rn(top, rule.c)), -SR_REF), SR_REF); };
    auto two_to = [](float n) { return __hiloint2double(max(1023 + (int)n, 0) << 20, 0); };  // n <= 0, 0 from -1023 on
    const bool online = has_p && rule.min_p == 0.0 && !rule.greedy;
    float tmax = -INFINITY, tref = -SR_REF;
    double tsum = 0.0;
    {
        // batches of SR_AHEAD vectors, the next one in flight while this one is looked at
        auto load = [&](int s, uint4 (&q)[SR_AHEAD]) {
            const int i0 = base + (s * 32 + lane) * E;
#pragma unroll
            for (int k = 0; k < SR_AHEAD; k++)
                q[k] = s + k < A.steps ? fetch(i0 + k * 32 * E) : make_uint4(~0u, ~0u, ~0u, ~0u);
        };
        float gm = -INFINITY;
        int g = 0, ahead = A.gsteps;  // the group, and its steps to come
        uint4 q[SR_AHEAD], nq[SR_AHEAD];
        load(0, q);
        for (int s = 0; s < A.steps; s += SR_AHEAD) {
            if (s + SR_AHEAD < A.steps) load(s + SR_AHEAD, nq);
            uint4 top4 = q[0];
#pragma unroll
            for (int k = 1; k < SR_AHEAD; k++) top4 = sr_max<T>(top4, q[k]);
            float m = -INFINITY;
            {
                float v[E];
                sr_unpack<T>(top4, v);
#pragma unroll
                for (int e = 0; e < E; e++) m = fmaxf(m, v[e]);
            }
            gm = fmaxf(gm, m);
            if (online && m > -INFINITY) {
                const float top_ref = ref(fmaxf(tmax, m));
                float sum[SR_AHEAD];
#pragma unroll
                for (int k = 0; k < SR_AHEAD; k++) {
                    float v[E];
                    // NaN and -inf as the lowest f32 or bf16, which weighs nothing at any T (fp16's would)
                    constexpr bool half = std::is_same<T, __half>::value;
                    sr_unpack<T>(half ? q[k] : sr_max<T>(q[k], sr_lowest<T>()), v);
                    sum[k] = 0.f;
#pragma unroll
                    for (int e = 0; e < E; e++)
                        sum[k] += ex2(__fmaf_rn(half ? fmaxf(v[e], -3.4028235e38f) : v[e], rule.c, -top_ref));
                }
                tsum = __fma_rn(tsum, two_to(tref - top_ref), (double)((sum[0] + sum[1]) + (sum[2] + sum[3])));
                tref = top_ref;
            }
            tmax = fmaxf(tmax, m);
            ahead -= SR_AHEAD;
            if (ahead <= 0 || s + SR_AHEAD >= A.steps) {
                gmax[g * SR_THREADS + tid] = gm;
                gm = -INFINITY;
                g++;
                ahead = A.gsteps;
            }
#pragma unroll
            for (int k = 0; k < SR_AHEAD; k++) q[k] = nq[k];
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
    auto push = [&](auto field, auto v) {  // own value into every rank's [rank]
        if (tid < cs) (cl.map_shared_rank(&S, tid)->*field)[rank] = v;
    };
    const float bmax = sr_reduce(tmax, reinterpret_cast<float *>(S.red), maxf);
    const float blow = sr_reduce(tmax > -INFINITY ? tmax : INFINITY, reinterpret_cast<float *>(S.red), minf);
    double bsum = 0.0;
    if (online)  // (relative to this CTA's ref)
        bsum = sr_reduce(__dmul_rn(tsum, two_to(tref - ref(bmax))), reinterpret_cast<double *>(S.red),
                         [](double a, double b) { return a + b; });
    if (cs > 1) csync();  // every rank has started
    push(&SrShared::max_of, bmax);
    push(&SrShared::low_of, blow);
    push(&SrShared::mass_of, bsum);
    csync();
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
        csync();
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
            const uint32_t kmax = sr_key(mx);
            uint32_t found = 0;
            for (int it = 0; it < 4 && !found; it++) {  // (the guess is an ulp or two off)
                const uint32_t k = k0 + lane - 16;
                const float v = sr_unkey(k);
                const uint32_t ok = __ballot_sync(0xffffffffu, v <= mx && rule.weight(v, mx, S.table) >= rule.min_p) |
                                    __ballot_sync(0xffffffffu, v > mx);
                if (ok && !(ok & 1)) found = k0 + __ffs(ok) - 1 - 16;
                k0 += ok ? -31 : 31;
            }
            if (!found && mx < INFINITY) {
                // The guess comes out of two large numbers next to 0, where f32 has many more between; or no difference
                // that f32 holds near the maximum counts at this T.  32 lanes close in.
                uint32_t l = sr_key(-INFINITY), h = kmax;  // never l, always h
                while (h - l > 1) {
                    const uint32_t k = l + (uint32_t)(((u64)(h - l) * (lane + 1)) >> 5);
                    const bool in = k >= h || (k > l && rule.weight(sr_unkey(k), mx, S.table) >= rule.min_p);
                    const int w = __ffs(__ballot_sync(0xffffffffu, in)) - 1;
                    const uint32_t nh = __shfl_sync(0xffffffffu, k, w), nl = __shfl_sync(0xffffffffu, k, max(w - 1, 0));
                    h = min(nh, h);
                    l = w > 0 ? nl : l;
                }
                found = h;
            }
            if (lane == 0) S.kmin = found ? found : kmax;
        }
        __syncthreads();
    }
    // survivors: x >= xmin (only the infinite logits weigh next to an infinite maximum)
    const float xmin = mx == INFINITY ? INFINITY : rule.min_p > 0.0 ? sr_unkey(S.kmin) : -3.4028235e38f;
    // The lowest f32 that weighs 2^-59 at least, and the lowest that weighs anything: e^-745.1332 is 2^-1075, which
    // binary64 rounds to 0.  (Rounded up: where f32 has no number between max - 41 T and the maximum, the next one below
    // is too small for vmin and does not stand for it.  From -FLT_MAX on at any T.)
    const float vmin = fmaxf(__double2float_ru((double)mx - 41.0 * rule.t), -3.4028235e38f);
    const float vzero = fmaxf(__double2float_ru((double)mx - 745.1332191019412 * rule.t), -3.4028235e38f);
    auto unit_of = [&](float v) -> u64 {
        if (mx == INFINITY) return v == mx ? (u64)SR_UNIT + 1 : 0;
        return v >= vzero ? (u64)rule.units_of(v, mx, vmin, S.table) : 0;  // (not NaN, not -inf)
    };
    // binary32 weight, relative error below 1e-5 wherever it is not negligible
    auto rough = [&](float v) {  // (of an infinite maximum: NaN's smaller one is 0, so 1 for an infinite logit)
        return ex2(fminf(__fmul_rn(__fsub_rn(v, mx), rule.c), 0.f));
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
    double m1 = 0.0;  // approximate mass of the survivors
    // (a maximum next to the lowest value, which the first pass took NaN and -inf for, or so many times T that f32 has
    // no place behind the point: the first pass's masses say nothing)
    // (T beyond what rule.c holds, or next to the logits' own size there: no approximate mass at all)
    const bool coarse =
        has_p && (rule.t >= 1e30 ? rule.t >= 1e36 || fabsf(mx) >= 1e20f : rule.t < 1.5e-30 && fabsf(mx) < 1e-18f);
    const bool summed = online && !coarse && mx > -1e38f && fabsf(__fmul_rn(mx, rule.c)) < SR_REF;
    // a rank's approximate mass, relative to the maximum's weight
    const float lift = summed ? ex2(__fmaf_rn(-mx, rule.c, ref(mx))) : 1.f;
    auto mass_at = [&](int i) {
        return summed ? S.mass_of[i] * two_to(ref(S.max_of[i]) - ref(mx)) * (double)lift : S.mass_of[i];
    };
    if (summed)
        for (int i = 0; i < cs; i++) m1 += mass_at(i);
    if (rule.min_p > 0.0) {
        few = true;
        if (!look_into([&](float m) { return m >= xmin; },
                       [&](float v, int i) {
                           if (v >= xmin) to_list(v, i);
                       }))
            too_many();
        // (too many of them, but none beyond top_k can stay: as without min-p)
        if (rule.top_k > 0 && rule.top_k <= SR_TOPK && !has_p) {
            csync();
            const bool over = lead->n_list > SR_LIST;
            csync();
            if (over) {
                if (rank == 0 && tid == 0) S.n_list = 0;
                few = false;
            }
        }
    }
    const bool then_topk = by_topk || (rule.min_p > 0.0 && !few);
    if (then_topk) {
        few = true;
        const float span = __fsub_rn(mx, low);
        const float inv = span > 0.f && span < INFINITY ? __fdiv_rn((float)(SR_BINS - 1), span) : 0.f;
        // (distances beyond the threads' lowest maximum share the last bin, which cannot be the threshold)
        auto bin = [&](float v) {
            return v == mx ? 0 : (int)fminf(__fmul_rn(__fsub_rn(mx, v), inv), (float)(SR_BINS - 1));
        };
        for (int g = 0; g < ngroups; g++) {
            const float m = gmax[g * SR_THREADS + tid];
            const int b = m > -INFINITY ? bin(m) : SR_BINS - 1;
            if (b < SR_BINS - 1) atomicAdd(&S.cnt[0][b], 1u);
        }
        csync();
        if (tid == 0) S.last_bin = SR_BINS;
        unsigned n[2] = {0, 0}, all;
        for (int i = 0; i < cs; i++) {
            const uint2 c2 = *reinterpret_cast<const uint2 *>(&cl.map_shared_rank(&S, i)->cnt[0][2 * tid]);
            n[0] += c2.x;
            n[1] += c2.y;
        }
        unsigned before = sr_scan(n[0] + n[1], reinterpret_cast<unsigned *>(S.red), &all);
#pragma unroll
        for (int k = 0; k < 2; k++) {
            if (before < (unsigned)rule.top_k && before + n[k] >= (unsigned)rule.top_k) S.last_bin = 2 * tid + k;
            before += n[k];
        }
        __syncthreads();
        const int last = S.last_bin;
        if (last < SR_BINS && inv > 0.f) {
            auto in = [&](float v) { return v >= xmin && bin(v) <= last; };
            if (!look_into(in, [&](float v, int i) {
                    if (in(v)) to_list(v, i);
                }))
                too_many();
        } else {
            few = false;  // fewer maxima than top_k, or equal ones
        }
    }

    auto value_of = [](u64 pr) { return sr_unkey((uint32_t)(pr >> 32)); };
    // Few entries: the block ranks them, a group of lanes adding up for one entry what counts() lets count.
    auto ranked = [&](int n, auto counts, auto use) {
        int g = 1;  // lanes an entry
        while (g < 32 && g * 2 * n <= SR_THREADS) g *= 2;
        const int c = tid / g;
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
    };
    // More: sorted, larger first(a, b) leading, then each thread's SR_EACH consecutive entries, with the mass before
    // them.  use(entry, its place, the mass before it, its own).
    auto sorted = [&](int n, auto larger, auto use) {
        int p = 2;
        while (p < n) p <<= 1;
        for (int i = n + tid; i < p; i += SR_THREADS) S.list[i] = 0;
        __syncthreads();
        for (int k = 2; k <= p; k <<= 1)
            for (int j = k >> 1; j > 0; j >>= 1) {
                for (int t = tid; t < p / 2; t += SR_THREADS) {
                    const int i = 2 * t - (t & (j - 1)), o = i + j;
                    const u64 a = S.list[i], b = S.list[o];
                    if (larger(b, a) == ((i & k) == 0)) {
                        S.list[i] = b;
                        S.list[o] = a;
                    }
                }
                __syncthreads();
            }
        u64 w[SR_EACH], sum = 0, all;
#pragma unroll
        for (int e = 0; e < SR_EACH; e++) {
            const int i = tid * SR_EACH + e;
            w[e] = i < n ? unit_of(value_of(S.list[i])) : 0;
            sum += w[e];
        }
        u64 before = sr_scan(sum, S.red, &all);
#pragma unroll
        for (int e = 0; e < SR_EACH; e++) {
            const int i = tid * SR_EACH + e;
            if (i < n) use(S.list[i], i, before, w[e]);
            before += w[e];
        }
    };
    // Where the cut falls in the list, with the mass and count above the list and the needed mass (its bounds lo, hi):
    // S.cut, its place S.first_bin, and of the list down to it S.kept_mass.  False where lo and hi do not agree.
    auto find_cut = [&](int n, u64 m_above, unsigned c_above, u64 lo, u64 hi) {
        if (tid == 0) S.first_bin = S.last_bin = n - 1;
        __syncthreads();
        int place[SR_EACH], k = 0;
        u64 upto[SR_EACH], pair[SR_EACH];
#pragma unroll
        for (int e = 0; e < SR_EACH; e++) place[e] = -1;
        auto look = [&](u64 mine, int number, u64 mass, u64 w) {
            const u64 run = m_above + mass + w;
            const bool full = rule.top_k && c_above + number + 1 >= (unsigned)rule.top_k;
            if (full || (has_p && run >= lo)) atomicMin(&S.first_bin, number);
            if (full || (has_p && run >= hi)) atomicMin(&S.last_bin, number);
#pragma unroll
            for (int e = 0; e < SR_EACH; e++)
                if (e == k) {
                    place[e] = number;
                    upto[e] = mass + w;
                    pair[e] = mine;
                }
            k++;
        };
        if (n <= SR_RANKED)
            ranked(n, [](u64 a, u64 b) { return a > b; },
                   [&](int c, u64 mine, int number, u64 mass) { look(mine, number, mass, S.wt[c]); });
        else
            sorted(n, [](u64 a, u64 b) { return a > b; }, look);
        __syncthreads();
        const int at = S.first_bin;
        if (at != S.last_bin) return false;
#pragma unroll
        for (int e = 0; e < SR_EACH; e++)
            if (place[e] == at) {
                S.cut = pair[e];
                S.kept_mass = upto[e];
            }
        __syncthreads();
        return true;
    };

    if (few) {
        csync();
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
                lo = summed ? rule.need((u64)(m1 * (1.0 - 4e-6) * SR_UNIT)) : 0;
                hi = summed ? rule.need((u64)(m1 * (1.0 + 4e-6) * SR_UNIT)) : ~0ull;
            } else if (has_p) {
                u64 m = 0;
                for (int i = tid; i < n; i += SR_THREADS) m += S.wt[i];
                lo = hi = rule.need(sr_reduce(m, S.red, addu));
            }
            if (!find_cut(n, 0, 0, lo, hi)) {
                u64 m = 0;  // the exact mass of the whole row
                const float from = fmaxf(xmin, vzero), top = fminf(mx, 3.4028235e38f);
                for (int i0 = tid * E; i0 < A.vocab; i0 += SR_AHEAD * SR_THREADS * E) {
                    uint4 q[SR_AHEAD];
#pragma unroll
                    for (int k = 0; k < SR_AHEAD; k++) q[k] = fetch(i0 + k * SR_THREADS * E);
#pragma unroll
                    for (int k = 0; k < SR_AHEAD; k++) {
                        float v[E];
                        sr_unpack<T>(q[k], v);
#pragma unroll
                        for (int e = 0; e < E; e++) {
                            const u64 w = rule.biased_units(v[e], top, vmin, S.table) - SR_BIAS;
                            m += v[e] >= from ? w : 0;
                        }
                    }
                }
                lo = rule.need(sr_reduce(m, S.red, addu));
                find_cut(n, 0, 0, lo, lo);
            }
            const u64 cut = S.cut, total = S.kept_mass;
            const u64 target = rule.place(total);
            // mass before each kept entry in index order (the low halves hold ~index)
            auto draw = [&](u64 mine, int, u64 mass, u64 w) {
                if (mass <= target && target < mass + w) {
                    A.tokens[row] = (int)~(uint32_t)mine;
                    if (A.probs)
                        A.probs[row] = (float)(rule.weight(value_of(mine), mx, S.table) * SR_UNIT / (double)total);
                }
            };
            if (n <= SR_RANKED)
                ranked(n, [&](u64 a, u64 b) { return a >= cut && (uint32_t)a > (uint32_t)b; },
                       [&](int c, u64 mine, int number, u64 mass) {
                           if (mine >= cut) draw(mine, number, mass, S.wt[c]);
                       });
            else
                sorted(S.first_bin + 1, [](u64 a, u64 b) { return (uint32_t)a > (uint32_t)b; }, draw);
            csync();  // the other ranks have read n_list before they left
            return;
        }
    }

    // ---- many candidates: the cut's range by bins of the distance to the maximum
    u64 cut = 0;  // the last kept (logit, index) pair
    // survivors from xa on stay, those in xb .. xa are the range that the cut lies in
    bool to_top = cuts;  // the range still reaches the maximum: xa is NaN, which nothing reaches
    float xa = cuts ? __int_as_float(0x7fffffff) : xmin, xb = xmin;
    auto side = [&](float v) { return v >= xa ? 1 : v >= xb ? 0 : -1; };
    // kept mass of every warp's run, to rank 0
    auto push_run = [&](u64 m) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
        if (lane == 0) lead->seg[rank * SR_WARPS + warp] = m;
    };
    unsigned c_above = 0, in_range = coarse ? SR_LIST + 1 : 0;
    if (cuts && !coarse) {
        // the approximate mass, where the first pass has not found it
        if (!summed) {
            double mass = 0.0;
            stream([&](float (&v)[E], int) {
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const float p = rough(v[e]);
                    sum += v[e] >= xmin ? p : 0.f;
                }
                mass += (double)sum;
            });
            mass = sr_reduce(mass, reinterpret_cast<double *>(S.red), [](double a, double b) { return a + b; });
            csync();  // the earlier values have been read
            push(&SrShared::mass_of, mass);
            for (int i = tid; i < SR_BINS; i += SR_THREADS) S.cnt[0][i] = 0;
            csync();
        } else if (then_topk) {
            csync();  // the counts have been read
            for (int i = tid; i < SR_BINS; i += SR_THREADS) S.cnt[0][i] = 0;
            __syncthreads();
        }
        if (!summed) {
            m1 = 0.0;
            for (int i = 0; i < cs; i++) m1 += S.mass_of[i];
        }
        // a rank's bins count its mass in units of 2^-31 of it (2^19 roundings of half a unit are 1.2e-4, the last bin's
        // 512 f32 additions 3e-5: below the slack)
        const float step = (float)mass_at(rank) * 0x1p-31f, per = step > 0.f ? __fdiv_rn(1.f, step) : 0.f;
        // The first round's bins reach to weights of 2^-43; with top-p no further than the weights that, all vocab of
        // them, would not make up what the cut leaves out.  The last bin holds the rest.
        float lo = 0.f, hi = __fdiv_rn(30.f, rule.c * 0.6931472f);
        if (has_p) {
            const float left = __fdiv_rn((float)A.vocab, __fmul_rn(fmaxf((float)(1.0 - rule.top_p), 1e-7f), (float)m1));
            hi = fminf(hi, __fdiv_rn(fmaxf(__log2f(left), 0.f) + 0.5f, rule.c));
        }
        float m_above = 0.f;
        for (int round = 0; round < SR_ROUNDS; round++) {
            const int buf = round & 1;
            const float width = hi - lo;
            const float inv = width > 0.f && width < INFINITY ? __fdiv_rn(1.f, width) : 0.f;
            const float from = __fsub_rn(mx, lo);
            auto bin = [&](float v) {  // (the low bits of 2^23 + bin; an infinite maximum's NaN saturates to 0)
                const float t = __saturatef(__fmul_rn(__fsub_rn(from, v), inv));
                return (int)(__float_as_uint(__fmaf_rd(t, (float)(SR_BINS - 1), 8388608.f)) - 0x4b000000u);
            };
            unsigned n_last = 0;  // (the last bin is a crowded one: counted in registers)
            float m_last = 0.f;
            stream([&](float (&v)[E], int) {
                int b[E];
                unsigned u[E];
                float m_here = 0.f;
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const float p = has_p ? rough(v[e]) : 0.f;
                    const int at = bin(v[e]);
                    b[e] = side(v[e]) == 0 ? at : SR_BINS;
                    m_here += b[e] == SR_BINS - 1 ? p : 0.f;
                    n_last += b[e] == SR_BINS - 1;
                    u[e] = __float2uint_rn(__fmul_rn(p, per));
                }
                m_last += m_here;
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (b[e] < SR_BINS - 1) {
                        atomicAdd(&S.cnt[buf][b[e]], 1u);
                        if (has_p) atomicAdd(&S.mass[buf][b[e]], u[e]);
                    }
            });
            n_last = sr_reduce(n_last, reinterpret_cast<unsigned *>(S.red),
                               [](unsigned a, unsigned b) { return a + b; });
            m_last = sr_reduce(m_last, reinterpret_cast<float *>(S.red), addf);
            if (tid == 0) {
                S.cnt[buf][SR_BINS - 1] = n_last;
                S.mass[buf][SR_BINS - 1] = __float2uint_rn(__fmul_rn(m_last, per));
            }
            csync();
            // this thread's bins 2 tid, 2 tid + 1: counts of all ranks, and of the ranks before this one
            unsigned n[2] = {0, 0}, n_low[2] = {0, 0}, n_all;
            float m[2] = {0.f, 0.f}, m_all;
            for (int i = 0; i < cs; i++) {
                const SrShared *o = cl.map_shared_rank(&S, i);
                const uint2 c2 = *reinterpret_cast<const uint2 *>(&o->cnt[buf][2 * tid]);
                if (i == rank) {
                    n_low[0] = n[0];
                    n_low[1] = n[1];
                }
                n[0] += c2.x;
                n[1] += c2.y;
                if (has_p) {
                    const uint2 m2 = *reinterpret_cast<const uint2 *>(&o->mass[buf][2 * tid]);
                    const float unit = (float)mass_at(i) * 0x1p-31f;
                    m[0] += __fmul_rn((float)m2.x, unit);
                    m[1] += __fmul_rn((float)m2.y, unit);
                }
            }
            unsigned nb = c_above + sr_scan(n[0] + n[1], reinterpret_cast<unsigned *>(S.red), &n_all);
            __syncthreads();
            float mb = m_above + sr_scan(m[0] + m[1], reinterpret_cast<float *>(S.red), &m_all);
            if (tid == 0) {
                S.first_bin = S.last_bin = SR_BINS;
                S.range_count = S.range_low = 0;
            }
            // (the buffer of the next round was read before this round's barrier)
            for (int i = tid; i < SR_BINS; i += SR_THREADS) S.cnt[buf ^ 1][i] = S.mass[buf ^ 1][i] = 0;
            __syncthreads();
            // the cut is in the first bin that may complete top_k or top_p, or behind it up to the first that must
            const float need = (float)(rule.top_p * m1), slack = 2e-4f * (float)m1;
            unsigned nb_of[2];
            float mb_of[2];
#pragma unroll
            for (int k = 0; k < 2; k++) {
                nb_of[k] = nb;
                mb_of[k] = mb;
                nb += n[k];
                mb += m[k];
                const bool full = rule.top_k && nb >= (unsigned)rule.top_k;
                if (n[k] && (full || (has_p && mb + slack >= need))) atomicMin(&S.first_bin, 2 * tid + k);
                if (n[k] && (full || (has_p && mb - slack >= need))) atomicMin(&S.last_bin, 2 * tid + k);
            }
            __syncthreads();
            const int fb = S.first_bin, lb = min(S.last_bin, SR_BINS - 1);
#pragma unroll
            for (int k = 0; k < 2; k++) {
                if (2 * tid + k >= fb && 2 * tid + k <= lb) {
                    atomicAdd(&S.range_count, n[k]);
                    atomicAdd(&S.range_low, n_low[k]);
                }
                if (2 * tid + k == fb) {
                    S.m_at = mb_of[k];
                    S.red[31] = nb_of[k];
                }
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
            // (the last bin reaches down to the lowest value of the type, a mask perhaps, and 512 distances tell nothing
            // apart there; and no finer bins divide what the masses' slack leaves open)
            if (in_range <= SR_LIST || lb >= SR_BINS - 1) break;
            // the next round divides these bins
            const float w1 = width * (1.f / (SR_BINS - 1));
            hi = lo + w1 * (lb + 1);
            lo = lo + w1 * fb;
        }
    }
    // ---- still more than the list holds: exact counts and masses of 512 bins of equal numbers of (key, index) pairs, 9
    // bits a pass, of whole keys as long as there is more than one; down to a list, or among equal logits to the cut
    bool found = false;
    if (in_range > SR_LIST) {
        constexpr int IB = 19;  // bits of an index
        static_assert(SR_MAX_VOCAB == 1 << IB, "a pair is a key and an index");
        auto place = [&](float v, int i) { return (u64)sr_key(v) << IB | (u64)(SR_MAX_VOCAB - 1 - i); };
        u64 m_above = 0, need = ~0ull;
        if (has_p) {
            u64 m = 0;
            stream([&](float (&v)[E], int) {
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const u64 w = v[e] >= xmin ? unit_of(v[e]) : 0;
                    m += w;
                    m_above += side(v[e]) > 0 ? w : 0;
                }
            });
            m = sr_reduce(m, S.red, addu);
            m_above = sr_reduce(m_above, S.red, addu);
            csync();  // (earlier uses of the slots are over)
            if (tid < cs) {
                SrShared *o = cl.map_shared_rank(&S, tid);
                o->slot[0][rank] = m;
                o->slot[1][rank] = m_above;
            }
            csync();
            m = m_above = 0;
            for (int i = 0; i < cs; i++) {
                m += S.slot[0][i];
                m_above += S.slot[1][i];
            }
            need = rule.need(m);
        }
        u64 top = (u64)(to_top ? sr_key(mx) : sr_key(xa) - 1) << IB | (SR_MAX_VOCAB - 1), low = (u64)sr_key(xb) << IB;
        for (;;) {
            const u64 span = top - low;
            const int bits = 64 - __clzll((long long)span), shift = max(bits - 9, span >> IB ? IB : 0);
            csync();  // the bins of the last pass have been read
            for (int i = tid; i < SR_BINS; i += SR_THREADS) S.cnt[0][i] = S.mass[0][i] = S.mass[1][i] = 0;
            __syncthreads();
            stream([&](float (&v)[E], int i) {
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const u64 at = place(v[e], i + e);
                    if (side(v[e]) != 0 || at > top || at < low) continue;
                    const int b = (int)((top - at) >> shift);
                    atomicAdd(&S.cnt[0][b], 1u);
                    if (has_p) {  // (two 32-bit atomics and the carry: a 64-bit one in shared memory is a loop)
                        const u64 w = unit_of(v[e]);
                        const unsigned w32 = (unsigned)w, sum = atomicAdd(&S.mass[0][b], w32) + w32;
                        atomicAdd(&S.mass[1][b], (unsigned)(w >> 32) + (sum < w32));
                    }
                }
            });
            if (tid == 0) S.first_bin = SR_BINS;
            csync();
            unsigned n[2] = {0, 0}, n_low[2] = {0, 0}, n_all;
            u64 m[2] = {0, 0}, all;
            for (int i = 0; i < cs; i++) {
                const SrShared *o = cl.map_shared_rank(&S, i);
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    if (i == rank) n_low[k] = n[k];
                    n[k] += o->cnt[0][2 * tid + k];
                    m[k] += (u64)o->mass[1][2 * tid + k] << 32 | o->mass[0][2 * tid + k];
                }
            }
            unsigned nb = c_above + sr_scan(n[0] + n[1], reinterpret_cast<unsigned *>(S.red), &n_all);
            __syncthreads();
            u64 mb = m_above + sr_scan(m[0] + m[1], S.red, &all);
            const unsigned nb0 = nb;
            const u64 mb0 = mb;
#pragma unroll
            for (int k = 0; k < 2; k++) {
                nb += n[k];
                mb += m[k];
                if (n[k] && ((rule.top_k && nb >= (unsigned)rule.top_k) || (has_p && mb >= need)))
                    atomicMin(&S.first_bin, 2 * tid + k);
            }
            __syncthreads();
            const int fb = S.first_bin;  // (the range holds the cut)
            if (fb >> 1 == tid) {
                const int k = fb & 1;
                S.range_count = k ? n[1] : n[0];
                S.range_low = k ? n_low[1] : n_low[0];
                S.red[31] = nb0 + (k ? n[0] : 0);
                S.target = mb0 + (k ? m[0] : 0);
            }
            __syncthreads();
            in_range = S.range_count;
            c_above = (unsigned)S.red[31];
            m_above = S.target;
            const u64 end = (u64)(fb + 1) << shift;
            if (end <= span) low = top - end + 1;
            top -= (u64)fb << shift;
            if (shift >= IB) {
                to_top = to_top && (uint32_t)(top >> IB) == sr_key(mx);
                if (!to_top) xa = sr_unkey((uint32_t)(top >> IB) + 1);
                xb = sr_unkey((uint32_t)(low >> IB));
                if (in_range <= SR_LIST) break;
            }
            if (shift == 0) {
                cut = (top >> IB) << 32 | (uint32_t)~(uint32_t)(SR_MAX_VOCAB - 1 - (int)(top & (SR_MAX_VOCAB - 1)));
                found = true;
                break;
            }
        }
    }
    // ---- exact masses: above the range (kept), and of all survivors where top-p needs it; the range to rank 0
    const bool listed = in_range > 0 && !found;
    const unsigned at0 = listed ? S.range_low : 0;  // the entries of the ranks before this one come first
    if (listed) {  // (in other cases a rank may still be reading rank 0's count)
        __syncthreads();
        if (tid == 0) S.n_list = 0;
        __syncthreads();
    }
    u64 kept = 0, m_all = 0;
    {
        // from which logit on they weigh and count (NaN: none does)
        const float none_of = __int_as_float(0x7fffffff);
        const float from_kept = xa == xa ? fmaxf(xa, vzero) : none_of, from_all = has_p ? fmaxf(xmin, vzero) : none_of;
        const float top = fminf(mx, 3.4028235e38f);
        stream([&](float (&v)[E], int i) {
            unsigned hits = 0;  // (no branch between the logits: their chains of double operations run together)
#pragma unroll
            for (int e = 0; e < E; e++) {
                const u64 w = rule.biased_units(v[e], top, vmin, S.table) - SR_BIAS;
                m_all += v[e] >= from_all ? w : 0;
                kept += v[e] >= from_kept ? w : 0;
                hits |= side(v[e]) == 0 ? 1u << e : 0u;
            }
            if (listed && hits)
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (hits >> e & 1u) lead->list[at0 + atomicAdd(&S.n_list, 1u)] = sr_pair(v[e], i + e);
        });
    }
    push_run(kept);
    m_all = sr_reduce(m_all, S.red, addu);
    if (tid == 0) lead->slot[1][rank] = m_all;
    csync();
    if (found) {
        stream([&](float (&v)[E], int i) {
#pragma unroll
            for (int e = 0; e < E; e++)
                if (side(v[e]) == 0 && sr_pair(v[e], i + e) >= cut) kept += unit_of(v[e]);
        });
        csync();  // the runs' masses have been read
        push_run(kept);
        csync();
    }
    if (rank != 0) return;
    // ---- rank 0 alone: the cut, the run that the draw falls into, the logit
    if (listed) {
        const int n = (int)in_range;
        for (int i = tid; i < n; i += SR_THREADS) S.wt[i] = unit_of(value_of(S.list[i]));
        u64 above = tid < cs * SR_WARPS ? S.seg[tid] : 0, mass = 0;
        above = sr_reduce(above, S.red, addu);
        for (int i = 0; i < cs; i++) mass += S.slot[1][i];
        const u64 need = has_p ? rule.need(mass) : ~0ull;
        find_cut(n, above, c_above, need, need);
        cut = S.cut;
        for (int i = tid; i < n; i += SR_THREADS)
            if (S.list[i] >= cut) {
                // (two 32-bit atomics and the carry: a 64-bit one in shared memory is a loop)
                const u64 w = unit_of(value_of(S.list[i]));
                unsigned *half = reinterpret_cast<unsigned *>(&S.seg[(int)~(uint32_t)S.list[i] / run]);
                const unsigned low32 = (unsigned)w, sum = atomicAdd(half, low32) + low32;
                atomicAdd(half + 1, (unsigned)(w >> 32) + (sum < low32));
            }
        __syncthreads();
    }
    const u64 mine = tid < cs * SR_WARPS ? S.seg[tid] : 0;
    if (tid == 0) S.where = 0;
    u64 total;
    const u64 before = sr_scan(mine, S.red, &total);
    u64 target = rule.place(total);
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
            upto += unit_of(v);
            if (upto > target) {
                A.tokens[row] = i;
                if (A.probs) A.probs[row] = (float)(rule.weight(v, mx, S.table) * SR_UNIT / (double)total);
                break;
            }
        }
    }
}

// CTAs a row: as many as still find a place at once (three CTAs an SM), while
// every lane keeps at least SR_AHEAD vectors.
template <typename T> static void launch_sample_rows(fb_ctx *ctx, SampleRowsArgs A, int64_t rows) {
    constexpr int step = SR_THREADS * SR_E<T>;  // logits of one step of a CTA
    int cs = 1;
    while (cs < SR_CLUSTER && rows * cs * 2 <= 3 * ctx->num_sms && A.vocab > cs * step * SR_AHEAD) cs *= 2;
    A.steps = (A.vocab + cs * step - 1) / (cs * step);
    A.chunk = A.steps * step;
    // groups of SR_AHEAD vectors, longer ones where a thread would have more than SR_GROUPS of them
    A.gsteps = SR_AHEAD * ((A.steps + SR_AHEAD * SR_GROUPS - 1) / (SR_AHEAD * SR_GROUPS));
    const size_t smem = (size_t)((A.steps + A.gsteps - 1) / A.gsteps) * SR_THREADS * 4;
    auto kernel = k_sample_rows<T>;
    // (the kernel's bound, not this call's size: the attribute belongs to the process, whose other threads launch other sizes)
    FB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SR_GROUPS * SR_THREADS * 4));
    if (cs > 8) FB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    launch_with(ctx->stream, false, kernel, dim3((unsigned)(rows * cs)), SR_THREADS, smem, (unsigned)cs, A);
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
