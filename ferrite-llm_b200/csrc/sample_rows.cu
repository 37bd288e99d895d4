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
// Bound: HBM (a row is read once, into the shared memory of a thread-block
// cluster); a few rows are bound by the cluster's steps.  No sort of the row:
//  * min-p: the threshold logit is found exactly (the f32 whose binary64 weight
//    is the first to reach min_p); the survivors are the candidates;
//  * top_k <= SR_TOPK: at least top_k of the threads' maxima lie above the
//    threshold that a 256-bin count of these maxima gives, so the cut does too:
//    the logits above it are the candidates (a little over top_k of them);
//  * otherwise: counts and approximate masses of 256 bins of the distance to
//    the maximum narrow the cut down to a range of at most SR_LIST logits, all
//    above it are kept.
// One CTA ranks the candidates against each other with exact weights (no sort:
// 512 at most, a few lanes each).  In the first two cases it draws from them
// alone and the cluster's other CTAs are gone by then.  A decision that leans on
// approximate masses is taken with their error on both sides; where that leaves
// it open, the exact mass of the row is summed.  Rows whose cut falls among more
// than SR_LIST logits that no bin tells apart are bisected by key.
#include <cooperative_groups.h>
#include <math.h>

#include <mutex>

#include "fb_internal.h"
#include "kq_common.cuh"

namespace fb {
namespace cg = cooperative_groups;

constexpr int SR_THREADS = 256;
constexpr int SR_WARPS = SR_THREADS / 32;
constexpr int SR_MAX_VOCAB = 1 << 19;
constexpr int SR_LIST = 512;    // candidates one CTA ranks
constexpr int SR_EACH = SR_LIST / SR_THREADS;
constexpr int SR_TOPK = 256;    // top_k up to here goes by the threads' maxima
constexpr int SR_BINS = 256;
constexpr int SR_CLUSTER = 16;
constexpr int SR_ROUNDS = 4;    // narrowings before the bisection
constexpr double SR_UNIT = 8796093022208.0;  // 2^43

using u64 = unsigned long long;

struct SampleRowsArgs {
    const void *logits;
    int64_t stride;
    int vocab, words;  // shared-memory words a thread (odd: its own run is free of bank conflicts)
    bool vec;          // rows start on 16 bytes
    const float *temperature, *top_p, *min_p, *uniform;
    const int32_t *top_k;
    int32_t *tokens;
    float *probs;
};

// A 32-bit word holds one f32 or two 16-bit logits.
template <typename T> struct SrWord;
template <> struct SrWord<float> {
    static constexpr int N = 1;
    static __device__ __forceinline__ void get(uint32_t w, float (&v)[1]) { v[0] = __uint_as_float(w); }
    static constexpr uint32_t PAD = 0x7fffffffu;  // NaN: never selected
};
template <> struct SrWord<__half> {
    static constexpr int N = 2;
    static __device__ __forceinline__ void get(uint32_t w, float (&v)[2]) {
        v[0] = __half2float(__ushort_as_half((unsigned short)w));
        v[1] = __half2float(__ushort_as_half((unsigned short)(w >> 16)));
    }
    static constexpr uint32_t PAD = 0x7fff7fffu;
};
template <> struct SrWord<__nv_bfloat16> {
    static constexpr int N = 2;
    static __device__ __forceinline__ void get(uint32_t w, float (&v)[2]) {
        v[0] = __uint_as_float(w << 16);
        v[1] = __uint_as_float(w & 0xffff0000u);
    }
    static constexpr uint32_t PAD = 0x7fff7fffu;
};

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
    double scale, min_p, top_p, t;  // scale = log2(e) 32 / T; min_p 0: off; top_p 2: off
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
        scale = 46.16624130844683 / t;  // 32 log2(e) / T
        c = (float)(scale * 0.03125);
        min_p = mp > 0.f ? fmin((double)mp, 1.0) : 0.0;
        top_p = tp < 1.f ? fmax((double)tp, 0.0) : 2.0;
        top_k = k > 0 && k < A.vocab ? k : 0;
        u = uu > 0.f ? fmin((double)uu, 1.0) : 0.0;
    }
    // exp((x - mx) / T) = 2^(z / 32), z = scale (x - mx): the table holds 2^(j / 32), and the rest |f| <= 1/2 of
    // a step is a Taylor polynomial of e^(f ln2 / 32) (argument below 0.011: degree 5 is below 2^-53).
    // The maximum itself (infinite too) weighs 1, NaN 0.
    __device__ __forceinline__ double weight(float x, float mx, const double *table) const {
        const double z = __dmul_rn((double)x - (double)mx, scale);
        const double y = fmax(z, -34400.0);  // 2^-1075 (NaN too)
        const double q = __dadd_rn(y, 6755399441055744.0);  // 1.5 * 2^52: the nearest integer in the low bits
        const int n = __double2loint(q);
        const double f = __dmul_rn(__dsub_rn(y, __dsub_rn(q, 6755399441055744.0)), 0.021660849392498290);  // ln2 / 32
        double p = __fma_rn(f, 1.0 / 120.0, 1.0 / 24.0);
        p = __fma_rn(p, f, 1.0 / 6.0);
        p = __fma_rn(p, f, 0.5);
        p = __fma_rn(p, f, 1.0);
        p = __fma_rn(p, f, 1.0);
        p = __dmul_rn(p, table[n & 31]);
        const int e = n >> 5, e0 = e / 2;  // (two factors: e reaches -1075; the second product rounds once)
        p = __dmul_rn(__dmul_rn(p, exp64_pow2(e0)), exp64_pow2(e - e0));
        return x == mx ? 1.0 : z > -34400.0 ? p : 0.0;
    }
    static __device__ __forceinline__ u64 units(double w) {
        if (!(w > 0.0)) return 0ull;
        // w 2^43 <= 2^43: adding 2^52 leaves its nearest integer in the low mantissa bits
        const u64 n = (u64)__double_as_longlong(__fma_rn(w, SR_UNIT, 4503599627370496.0)) & 0xfffffffffffffull;
        return n ? n : 1ull;
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
    u64 list[SR_LIST], wt[SR_LIST];    // rank 0: the candidates and their weights
    u64 slot[2][SR_CLUSTER];           // pushed by every rank
    u64 red[32];
    double table[32];
    float max_of[SR_CLUSTER], low_of[SR_CLUSTER], mass_of[SR_CLUSTER];
    float unit_of[SR_CLUSTER];         // weight of one step of a rank's mass bins
    uint32_t cnt[2][SR_BINS], mass[2][SR_BINS];
    u64 cut;                           // pushed by rank 0
    u64 kept_mass;
    unsigned n_list;                   // rank 0: candidates pushed
    int first_bin, last_bin;
    unsigned range_low;
    uint32_t kmin;
    unsigned range_count;
};

__device__ __forceinline__ float sr_load(const float *p, int i) { return p[i]; }
__device__ __forceinline__ float sr_load(const __half *p, int i) { return __half2float(p[i]); }
__device__ __forceinline__ float sr_load(const __nv_bfloat16 *p, int i) { return __bfloat162float(p[i]); }

static_assert(SR_BINS == SR_THREADS, "a thread a bin");
template <typename T> __global__ void __launch_bounds__(SR_THREADS, 4) k_sample_rows(const SampleRowsArgs A) {
    using W = SrWord<T>;
    constexpr int N = W::N;
    extern __shared__ __align__(16) uint32_t xs[];
    __shared__ SrShared S;
    cg::cluster_group cl = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, rank = cl.block_rank(), cs = cl.num_blocks();
    const int64_t row = blockIdx.x / cs;
    const int nwords = SR_THREADS * A.words, base = rank * nwords * N;  // this CTA's logits: base .. base + nwords * N - 1
    const T *x = static_cast<const T *>(A.logits) + row * A.stride;
    RowRule rule;
    rule.load(A, row);
    auto addu = [](u64 a, u64 b) { return a + b; };

    // ---- the row into shared memory; every thread's maximum of what it loads
    float tmax = -INFINITY;
    if (tid < 32) S.table[tid] = exp2((double)tid * 0.03125);
    if (tid == 0) S.n_list = 0;
    for (int i = tid; i < SR_BINS; i += SR_THREADS) S.cnt[0][i] = S.mass[0][i] = 0;
    if (A.vec) {
        constexpr int E = 4 * N;
#pragma unroll 5
        for (int v = tid; v < nwords / 4; v += SR_THREADS) {
            const int i = base + v * E;
            uint4 q = make_uint4(W::PAD, W::PAD, W::PAD, W::PAD);
            if (i + E <= A.vocab) {
                q = __ldg(reinterpret_cast<const uint4 *>(x + i));
            } else if (i < A.vocab) {
                T *e = reinterpret_cast<T *>(&q);
                for (int k = 0; i + k < A.vocab; k++) e[k] = x[i + k];
            }
            reinterpret_cast<uint4 *>(xs)[v] = q;
            const uint32_t w4[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int k = 0; k < 4; k++) {
                float f[N];
                W::get(w4[k], f);
#pragma unroll
                for (int e = 0; e < N; e++) tmax = fmaxf(tmax, f[e]);
            }
        }
    } else {
#pragma unroll 4
        for (int v = tid; v < nwords; v += SR_THREADS) {
            uint32_t q = W::PAD;
            T *e = reinterpret_cast<T *>(&q);
#pragma unroll
            for (int k = 0; k < N; k++)
                if (base + v * N + k < A.vocab) e[k] = x[base + v * N + k];
            xs[v] = q;
            float f[N];
            W::get(q, f);
#pragma unroll
            for (int k = 0; k < N; k++) tmax = fmaxf(tmax, f[k]);
        }
    }
    // f(logit, index) over the logits that a lane's threads of this warp loaded, for the lanes whose flag is set: the
    // whole warp looks through one lane's logits at a time
    auto loaded = [&](bool flag, auto f) {
        for (uint32_t todo = __ballot_sync(0xffffffffu, flag); todo; todo &= todo - 1) {
            const int src = (tid & ~31) + __ffs(todo) - 1;
            for (int q = lane; q < ((A.words + 3) & ~3); q += 32) {
                const int v = A.vec ? 4 * (src + SR_THREADS * (q >> 2)) + (q & 3) : src + SR_THREADS * q;
                if (v >= nwords) continue;
                float g[N];
                W::get(xs[v], g);
#pragma unroll
                for (int k = 0; k < N; k++) f(g[k], base + v * N + k);
            }
        }
    };
    // f(logit, index) over this thread's run of consecutive logits
    auto own = [&](auto f) {
#pragma unroll 4
        for (int j = 0; j < A.words; j++) {
            const int v = tid * A.words + j;
            float q[N];
            W::get(xs[v], q);
#pragma unroll
            for (int k = 0; k < N; k++) f(q[k], base + v * N + k);
        }
    };
    auto push = [&](float (SrShared::*field)[SR_CLUSTER], float v) {  // own value into every rank's [rank]
        if (tid < cs) (cl.map_shared_rank(&S, tid)->*field)[rank] = v;
    };
    auto maxf = [](float a, float b) { return fmaxf(a, b); };
    auto minf = [](float a, float b) { return fminf(a, b); };
    const float bmax = sr_reduce(tmax, reinterpret_cast<float *>(S.red), maxf);
    const float blow = sr_reduce(tmax > -INFINITY ? tmax : INFINITY, reinterpret_cast<float *>(S.red), minf);
    cl.sync();  // every rank has started
    push(&SrShared::max_of, bmax);
    push(&SrShared::low_of, blow);
    cl.sync();
    float mx = -INFINITY, low = INFINITY;  // the largest logit, the lowest of the threads' finite maxima
    for (int i = 0; i < cs; i++) {
        mx = fmaxf(mx, S.max_of[i]);
        low = fminf(low, S.low_of[i]);
    }
    if (rule.greedy || mx == -INFINITY) {
        // the first of the largest logits (a row of -inf has one, a row of NaN none)
        u64 first = ~0ull;
        if (rule.greedy)
            loaded(tmax == mx, [&](float v, int i) {
                if (v == mx) first = min(first, (u64)i);
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
    const bool by_topk = rule.top_k > 0 && rule.top_k <= SR_TOPK;
    const bool has_p = rule.top_p < 1.0, cuts = rule.top_k > 0 || has_p;
    auto unit_of = [&](float v) { return RowRule::units(rule.weight(v, mx, S.table)); };
    // binary32 weight, relative error below 1e-5 wherever it is not negligible
    auto rough = [&](float v) {
        float e;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(__fmul_rn(__fsub_rn(v, mx), rule.c)));
        return v == mx ? 1.f : mx == INFINITY ? 0.f : e;
    };
    auto rough_mass = [&]() {  // of this CTA's survivors
        float m = 0.f;
#pragma unroll 4
        for (int v = tid; v < nwords; v += SR_THREADS) {
            float q[N];
            W::get(xs[v], q);
#pragma unroll
            for (int k = 0; k < N; k++) {
                const float e = rough(q[k]);
                m += q[k] >= xmin ? e : 0.f;
            }
        }
        return sr_reduce(m, reinterpret_cast<float *>(S.red), [](float a, float b) { return a + b; });
    };

    // ---- few candidates: min-p's survivors, or what lies above the threads' top_k-th largest maximum
    SrShared *lead = cl.map_shared_rank(&S, 0);
    auto to_list = [&](float v, int i) {
        const unsigned at = atomicAdd(&lead->n_list, 1u);
        if (at < SR_LIST) lead->list[at] = sr_pair(v, i);
    };
    bool few = false;
    float m1 = 0.f;  // approximate mass of the survivors
    if (rule.min_p > 0.0) {
        few = true;
        loaded(tmax >= xmin, [&](float v, int i) {
            if (v >= xmin) to_list(v, i);
        });
    } else if (by_topk) {
        few = true;
        const float span = __fsub_rn(mx, low);
        const float inv = span > 0.f && span < INFINITY ? __fdiv_rn((float)(SR_BINS - 1), span) : 0.f;
        auto bin = [&](float v) { return v == mx ? 0 : (int)fminf(__fmul_rn(__fsub_rn(mx, v), inv), (float)SR_BINS); };
        if (tmax > -INFINITY) atomicAdd(&S.cnt[0][min(bin(tmax), SR_BINS - 1)], 1u);
        if (has_p) {
            const float m = rough_mass();
            push(&SrShared::mass_of, m);
        }
        cl.sync();
        if (tid == 0) S.last_bin = SR_BINS;
        unsigned n = 0, all;
        for (int i = 0; i < cs; i++) n += cl.map_shared_rank(&S, i)->cnt[0][tid];
        const unsigned before = sr_scan(n, reinterpret_cast<unsigned *>(S.red), &all);
        if (before < (unsigned)rule.top_k && before + n >= (unsigned)rule.top_k) S.last_bin = tid;
        __syncthreads();
        const int last = S.last_bin;
        for (int i = 0; i < cs; i++) m1 += has_p ? S.mass_of[i] : 0.f;
        if (last < SR_BINS && inv > 0.f) {
            loaded(tmax > -INFINITY && bin(tmax) <= last, [&](float v, int i) {
                if (v > -INFINITY && bin(v) <= last) to_list(v, i);
            });
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
            // the other ranks have read n_list before they left
            cl.sync();
            return;
        }
    }

    // ---- many candidates: the cut's range by bins of the distance to the maximum
    u64 cut = 0;  // the last kept (logit, index) pair
    u64 kept_sum = 0;  // this thread's mass that is certainly kept
    float d0[SR_ROUNDS] = {}, inv[SR_ROUNDS] = {};
    int b0[SR_ROUNDS] = {}, b1[SR_ROUNDS] = {};
    int rounds = 0;
    // where a survivor lies: 1 above the range (kept), 0 inside, -1 below
    auto dist = [&](float v) { return v == mx ? 0.f : __fsub_rn(mx, v); };
    auto bin_in = [&](float d, int r) {
        return (int)fminf(fmaxf(__fmul_rn(__fsub_rn(d, d0[r]), inv[r]), 0.f), (float)(SR_BINS - 1));
    };
    auto side = [&](float v) {
        const float d = dist(v);
#pragma unroll
        for (int r = 0; r < SR_ROUNDS; r++) {
            if (r >= rounds) break;
            const int b = bin_in(d, r);
            if (b < b0[r]) return 1;
            if (b > b1[r]) return -1;
        }
        return 0;
    };
    if (cuts) {
        // lowest survivor, and the approximate mass
        float lw = INFINITY, mass = 0.f;
#pragma unroll 4
        for (int v = tid; v < nwords; v += SR_THREADS) {
            float q[N];
            W::get(xs[v], q);
#pragma unroll
            for (int k = 0; k < N; k++) {
                const bool in = q[k] >= xmin;
                lw = in ? fminf(lw, q[k]) : lw;
                const float e = rough(q[k]);
                mass += in ? e : 0.f;
            }
        }
        lw = sr_reduce(lw, reinterpret_cast<float *>(S.red), minf);
        mass = sr_reduce(mass, reinterpret_cast<float *>(S.red), [](float a, float b) { return a + b; });
        const float step = mass > 0.f ? __fmul_rn(mass, 0x1p-30f) : 0.f;
        cl.sync();  // the earlier slots have been read
        push(&SrShared::low_of, lw);
        push(&SrShared::mass_of, mass);
        push(&SrShared::unit_of, step);
        for (int i = tid; i < SR_BINS; i += SR_THREADS) S.cnt[0][i] = S.mass[0][i] = 0;
        cl.sync();
        low = INFINITY;
        m1 = 0.f;
        for (int i = 0; i < cs; i++) {
            low = fminf(low, S.low_of[i]);
            m1 += S.mass_of[i];
        }
        const float per = step > 0.f ? __fdiv_rn(1.f, step) : 0.f;
        // weights below 2^-43 share the last bin of the first round
        float lo = 0.f, hi = fminf(dist(low), __fdiv_rn(30.f, rule.c * 0.6931472f));
        unsigned c_above = 0, in_range = 0;
        float m_above = 0.f;
        for (; rounds < SR_ROUNDS; rounds++) {
            const int buf = rounds & 1;
            const float width = hi - lo;
#pragma unroll
            for (int r = 0; r < SR_ROUNDS; r++)  // (fixed indexes: the rounds stay in registers)
                if (r == rounds) {
                    d0[r] = lo;
                    inv[r] = width > 0.f && width < INFINITY ? __fdiv_rn((float)(SR_BINS - 1), width) : 0.f;
                }
            own([&](float v, int) {
                if (!(v >= xmin) || side(v) != 0) return;
                int b = 0;
#pragma unroll
                for (int r = 0; r < SR_ROUNDS; r++)
                    if (r == rounds) b = bin_in(dist(v), r);
                atomicAdd(&S.cnt[buf][b], 1u);
                if (has_p) atomicAdd(&S.mass[buf][b], __float2uint_rn(__fmul_rn(rough(v), per)));
            });
            cl.sync();
            unsigned n = 0, n_low = 0, n_all;  // n_low: of the ranks before this one
            float m = 0.f, m_all;
            for (int i = 0; i < cs; i++) {
                const SrShared *o = cl.map_shared_rank(&S, i);
                if (i == rank) n_low = n;
                n += o->cnt[buf][tid];
                if (has_p) m += __fmul_rn((float)o->mass[buf][tid], S.unit_of[i]);
            }
            const unsigned nb = c_above + sr_scan(n, reinterpret_cast<unsigned *>(S.red), &n_all);
            __syncthreads();
            const float mb = m_above + sr_scan(m, reinterpret_cast<float *>(S.red), &m_all);
            // the cut is in the first bin that may complete top_k or top_p, or behind it up to the first that must
            const float need = (float)rule.top_p * m1, slack = 2e-4f * m1;
            const bool full = rule.top_k && nb + n >= (unsigned)rule.top_k;
            const bool may = n && (full || (has_p && mb + m + slack >= need)), must = n && (full || (has_p && mb + m - slack >= need));
            if (tid == 0) {
                S.first_bin = S.last_bin = SR_BINS;
                S.range_count = S.range_low = 0;
            }
            // (the buffer of the next round was read before this round's barrier)
            for (int i = tid; i < SR_BINS; i += SR_THREADS) S.cnt[buf ^ 1][i] = S.mass[buf ^ 1][i] = 0;
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
                S.max_of[0] = mb;  // (the maxima have been read)
                S.red[31] = nb;
            }
            __syncthreads();
            in_range = fb < SR_BINS ? S.range_count : 0;
#pragma unroll
            for (int r = 0; r < SR_ROUNDS; r++)
                if (r == rounds) {
                    b0[r] = fb;
                    b1[r] = lb;
                }
            if (fb >= SR_BINS) {  // nothing completes them: all survivors of this range stay
                in_range = 0;
                rounds++;
                break;
            }
            c_above = (unsigned)S.red[31];
            m_above = S.max_of[0];
            if (in_range <= SR_LIST) {
                rounds++;
                break;
            }
            // the next round divides these bins
            const float w1 = width * (1.f / (SR_BINS - 1));
            const float nlo = lo + w1 * fb, nhi = lb >= SR_BINS - 1 ? fmaxf(dist(low), hi) : lo + w1 * (lb + 1);
            lo = nlo;
            hi = nhi;
        }
        // ---- exact masses: above the range (kept), and of all survivors where top-p needs it; the range to rank 0
        const bool listed = in_range > 0 && in_range <= SR_LIST;
        const unsigned at0 = S.range_low;  // the entries of the ranks before this one come first
        __syncthreads();
        if (tid == 0) S.n_list = 0;
        __syncthreads();
        u64 m_all = 0;
        own([&](float v, int i) {
            const int s = v >= xmin ? side(v) : -1;
            u64 w = 0;
            if (has_p || s > 0) w = unit_of(v);
            m_all += v >= xmin ? w : 0;
            kept_sum += s > 0 ? w : 0;
            if (s == 0 && listed) lead->list[at0 + atomicAdd(&S.n_list, 1u)] = sr_pair(v, i);
        });
        const u64 above = sr_reduce(kept_sum, S.red, addu), all = sr_reduce(m_all, S.red, addu);
        if (tid < cs) {
            SrShared *o = cl.map_shared_rank(&S, tid);
            o->slot[0][rank] = above;
            o->slot[1][rank] = all;
        }
        cl.sync();
        u64 above_all = 0, mass_all = 0;
        for (int i = 0; i < cs; i++) {
            above_all += S.slot[0][i];
            mass_all += S.slot[1][i];
        }
        const u64 need = has_p ? need_of((double)mass_all) : ~0ull;
        if (in_range == 0) {
            cut = 0;  // every survivor down to the range's end
        } else if (listed) {
            if (rank == 0) {
                const int n = (int)in_range;
                for (int i = tid; i < n; i += SR_THREADS) S.wt[i] = unit_of(value_of(S.list[i]));
                __syncthreads();
                find_cut(n, above_all, c_above, need, need);
                if (tid < cs) cl.map_shared_rank(&S, tid)->cut = S.cut;
            }
            cl.sync();
            cut = S.cut;
        } else {
            // bisection over (key, index) pairs: the largest pair whose upper set completes top_k or top_p
            u64 lo_pair = 0, hi_pair = ~0ull;
            while (hi_pair - lo_pair > 1) {
                const u64 mid = lo_pair + (hi_pair - lo_pair) / 2;
                u64 m = 0, n = 0;
                own([&](float v, int i) {
                    if (v >= xmin && side(v) == 0 && sr_pair(v, i) >= mid) {
                        n++;
                        if (has_p) m += unit_of(v);
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
                m = above_all;
                n = c_above;
                for (int i = 0; i < cs; i++) {
                    m += S.slot[0][i];
                    n += S.slot[1][i];
                }
                if ((rule.top_k && n >= (u64)rule.top_k) || (has_p && m >= need && m > 0)) lo_pair = mid;
                else hi_pair = mid;
            }
            cut = lo_pair;
        }
        // what stays inside the range
        if (in_range)
            own([&](float v, int i) {
                if (v >= xmin && side(v) == 0 && sr_pair(v, i) >= cut) kept_sum += unit_of(v);
            });
    } else {
        own([&](float v, int) {
            if (v >= xmin) kept_sum += unit_of(v);
        });
    }
    // ---- the draw, in index order: ranks, threads, logits
    u64 mine;
    const u64 before = sr_scan(kept_sum, S.red, &mine);
    cl.sync();  // the slots have been read
    if (tid < cs) cl.map_shared_rank(&S, tid)->slot[0][rank] = mine;
    cl.sync();
    u64 total = 0, lower = 0;
    for (int i = 0; i < cs; i++) {
        if (i < rank) lower += S.slot[0][i];
        total += S.slot[0][i];
    }
    u64 target = (u64)(rule.u * (double)total);
    if (target >= total) target = total - 1;
    u64 run = lower + before;
    if (run <= target && target < run + kept_sum) {
        bool found = false;
        own([&](float v, int i) {
            if (found || !(v >= xmin)) return;
            const int s = cuts ? side(v) : 1;
            if (s < 0 || (s == 0 && sr_pair(v, i) < cut)) return;
            const double w = rule.weight(v, mx, S.table);
            run += RowRule::units(w);
            if (run > target) {
                found = true;
                A.tokens[row] = i;
                if (A.probs) A.probs[row] = (float)(w * SR_UNIT / (double)total);
            }
        });
    }
}

// CTAs a row: as many as bring its logits below SR_CHUNK bytes of shared
// memory a CTA (four CTAs an SM, so that one's steps hide another's), and more
// while SMs would stay empty and every thread keeps eight logits.
constexpr int SR_CHUNK = 48 * 1024;
template <typename T> static void launch_sample_rows(fb_ctx *ctx, SampleRowsArgs A, int64_t rows) {
    const int64_t bytes = (int64_t)A.vocab * (int64_t)sizeof(T);
    int cs = 1;
    while (cs < SR_CLUSTER && bytes > (int64_t)cs * SR_CHUNK) cs *= 2;
    while (cs < SR_CLUSTER && rows * cs * 2 <= ctx->num_sms && A.vocab >= 2 * cs * SR_THREADS * 8) cs *= 2;
    const int64_t words = (bytes + 3) / 4;
    A.words = (int)((words + (int64_t)cs * SR_THREADS - 1) / ((int64_t)cs * SR_THREADS)) | 1;
    const size_t smem = (size_t)SR_THREADS * A.words * 4;
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
