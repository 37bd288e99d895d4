// One token per logits row from given random numbers (fb_sample_rows): the
// rules of the reference sampler (crates/ferrite-core/src/sampling.rs:61-239)
// for many rows with settings of their own, without its host round trip.
//
// Mathematics: w_i = exp((x_i - max) / T).  In the row sorted by descending
// logit (equal logits in index order) min-p, top-p and top-k each keep a
// prefix, so the kept set is the shortest of the three: all logits above a
// cut key and the first few equal to it.  The cut is the largest key whose
// upper set holds top_k tokens or top_p of the mass.  Masses are 64-bit
// integers in units of 2^-43 (vocab <= 2^19 keeps them below 2^62), summed in
// any order with one result; a weight that is not zero counts for one unit at
// least, so no kept token is unreachable.
#include <math.h>

#include "fb_internal.h"
#include "kq_common.cuh"

namespace fb {

constexpr int SR_THREADS = 1024;
constexpr int SR_MAX_VOCAB = 1 << 19;

struct SampleRowsArgs {
    const void *logits;
    int64_t stride;
    int vocab;
    const float *temperature, *top_p, *min_p, *uniform;
    const int32_t *top_k;
    int32_t *tokens;
    float *probs;
};

__device__ __forceinline__ float sr_load(const float *p, int i) { return p[i]; }
__device__ __forceinline__ float sr_load(const __half *p, int i) { return __half2float(p[i]); }
__device__ __forceinline__ float sr_load(const __nv_bfloat16 *p, int i) { return __bfloat162float(p[i]); }

// Order-preserving key of a logit (-0 as +0); 0 for NaN, which sorts below all.
__device__ __forceinline__ uint32_t sr_key(float x) {
    if (x != x) return 0u;
    const uint32_t b = __float_as_uint(__fadd_rn(x, 0.f));
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

// A row's settings.
struct RowRule {
    double inv_t, min_p, top_p;  // min_p 0: off; top_p 2: off
    int top_k;                   // 0: off
    double u;
    bool greedy;
    __device__ __forceinline__ void load(const SampleRowsArgs &A, int64_t r) {
        const float t = A.temperature ? A.temperature[r] : 1.f;
        greedy = t <= 0.f;
        inv_t = (t != t || greedy) ? 1.0 : 1.0 / (double)t;
        const float mp = A.min_p ? A.min_p[r] : 0.f, tp = A.top_p ? A.top_p[r] : 1.f, uu = A.uniform[r];
        min_p = mp > 0.f ? fmin((double)mp, 1.0) : 0.0;
        top_p = tp < 1.f ? fmax((double)tp, 0.0) : 2.0;
        const int k = A.top_k ? A.top_k[r] : 0;
        top_k = k > 0 && k < A.vocab ? k : 0;
        u = uu > 0.f ? fmin((double)uu, 1.0) : 0.0;
    }
    // exp((x - mx) / T); the maximum itself (infinite too) weighs 1
    __device__ __forceinline__ double weight(float x, float mx) const {
        if (x == mx) return 1.0;
        const double d = (double)x - (double)mx;
        return d < 0.0 ? exp64(__dmul_rn(d, inv_t)) : 0.0;  // NaN: 0
    }
};
__device__ __forceinline__ unsigned long long sr_units(double w) {
    if (!(w > 0.0)) return 0ull;
    const unsigned long long n = (unsigned long long)__double2ull_rn(__dmul_rn(w, 8796093022208.0));  // 2^43
    return n ? n : 1ull;
}

template <typename V, typename Op> __device__ __forceinline__ V sr_reduce(V v, V *sh, Op op) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    V r = sh[0];
    for (int w = 1; w < SR_THREADS / 32; w++) r = op(r, sh[w]);
    return r;
}

template <typename T> __global__ void __launch_bounds__(SR_THREADS) k_sample_rows(SampleRowsArgs A) {
    using u64 = unsigned long long;
    __shared__ u64 sh[32];
    __shared__ u64 scan[SR_THREADS];
    __shared__ int pick;
    const int64_t r = blockIdx.x;
    const T *x = static_cast<const T *>(A.logits) + r * A.stride;
    RowRule rule;
    rule.load(A, r);
    auto maxu = [](u64 a, u64 b) { return a > b ? a : b; };
    auto add = [](u64 a, u64 b) { return a + b; };
    // the largest logit, the first of equal ones: key, then the reversed index
    u64 best = 0;
    for (int i = threadIdx.x; i < A.vocab; i += SR_THREADS) {
        const uint32_t k = sr_key(sr_load(x, i));
        if (k) best = maxu(best, ((u64)k << 32) | (uint32_t)(0x7fffffff - i));
    }
    best = sr_reduce(best, sh, maxu);
    const int first = 0x7fffffff - (int)(uint32_t)best;
    const float mx = best ? sr_load(x, first) : 0.f;
    if (!best || rule.greedy || mx == -INFINITY) {
        if (threadIdx.x == 0) {
            const bool none = !best || !rule.greedy;
            A.tokens[r] = none ? -1 : first;
            if (A.probs) A.probs[r] = none ? 0.f : 1.f;
        }
        return;
    }
    auto units = [&](float v) -> u64 {  // 0 where min-p (or NaN) leaves the token out
        const double w = rule.weight(v, mx);
        return w >= rule.min_p ? sr_units(w) : 0ull;
    };
    // the cut: the largest key whose upper set holds top_k tokens or top_p of the min-p mass
    u64 mass = 0;
    for (int i = threadIdx.x; i < A.vocab; i += SR_THREADS) mass += units(sr_load(x, i));
    mass = sr_reduce(mass, sh, add);
    const u64 need = rule.top_p < 1.0 ? (u64)ceil(rule.top_p * (double)mass) : ~0ull;
    const u64 kk = rule.top_k ? (u64)rule.top_k : ~0ull;
    uint32_t lo = 0, hi = 0xffffffffu;  // holds(lo) taken as true, holds(hi) false
    u64 m_above = 0, c_above = 0;
    while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        u64 m = 0, c = 0;
        for (int i = threadIdx.x; i < A.vocab; i += SR_THREADS) {
            const float v = sr_load(x, i);
            if (sr_key(v) >= mid) {
                const u64 w = units(v);
                m += w;
                c += w != 0;
            }
        }
        m = sr_reduce(m, sh, add);
        c = sr_reduce(c, sh, add);
        if ((m >= need && m > 0) || c >= kk) lo = mid;
        else {
            hi = mid;
            m_above = m;
            c_above = c;
        }
    }
    // how many of the tokens at the cut (all of one weight) stay
    u64 ties = ~0ull;
    if (lo > 0) {
        const float vcut = __uint_as_float((lo & 0x80000000u) ? lo & 0x7fffffffu : ~lo);
        const u64 wcut = units(vcut);
        if (kk != ~0ull && c_above < kk) ties = kk - c_above;
        if (need != ~0ull && wcut) {
            const u64 lack = need > m_above ? need - m_above : 0ull;
            const u64 t = lack ? (lack + wcut - 1) / wcut : 1ull;
            ties = ties < t ? ties : t;
        }
    }
    // contiguous ranges in index order: first the ties before each, then the mass
    const int per = (A.vocab + SR_THREADS - 1) / SR_THREADS;
    const int i0 = min(A.vocab, (int)threadIdx.x * per), i1 = min(A.vocab, i0 + per);
    auto exclusive = [&](u64 v) {
        __syncthreads();
        scan[threadIdx.x] = v;
        __syncthreads();
        for (int o = 1; o < SR_THREADS; o <<= 1) {
            const u64 y = threadIdx.x >= o ? scan[threadIdx.x - o] : 0;
            __syncthreads();
            scan[threadIdx.x] += y;
            __syncthreads();
        }
        return scan[threadIdx.x] - v;
    };
    u64 eq = 0;
    for (int i = i0; i < i1; i++) eq += sr_key(sr_load(x, i)) == lo;
    const u64 eq0 = exclusive(eq);
    auto walk = [&](auto f) {  // kept units in index order
        u64 e = eq0;
        for (int i = i0; i < i1; i++) {
            const float v = sr_load(x, i);
            const uint32_t k = sr_key(v);
            const bool keep = k > lo || (k == lo && lo > 0 && e < ties);
            e += k == lo;
            if (keep && f(i, units(v))) break;
        }
    };
    u64 part = 0;
    walk([&](int, u64 w) {
        part += w;
        return false;
    });
    const u64 before = exclusive(part);
    const u64 total = scan[SR_THREADS - 1];
    u64 target = (u64)(rule.u * (double)total);
    if (target >= total) target = total - 1;
    if (threadIdx.x == 0) pick = -1;
    __syncthreads();
    if (before <= target && target < before + part) {
        u64 run = before;
        walk([&](int i, u64 w) {
            run += w;
            if (run > target) {
                pick = i;
                return true;
            }
            return false;
        });
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        A.tokens[r] = pick;
        // the weight itself, not its units: a far token drawn by u = 0 keeps its probability
        if (A.probs) A.probs[r] = (float)(rule.weight(sr_load(x, pick), mx) * 8796093022208.0 / (double)total);
    }
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
        FB_REQUIRE(((uintptr_t)logits_dev & (dtype == FB_F32 ? 3 : 1)) == 0 &&
                       (((uintptr_t)temperature_dev | (uintptr_t)top_k_dev | (uintptr_t)top_p_dev |
                         (uintptr_t)min_p_dev | (uintptr_t)uniform_dev | (uintptr_t)tokens_dev |
                         (uintptr_t)probs_dev) & 3) == 0,
                   "sample_rows: misaligned pointer");
        DeviceGuard guard(ctx->device);
        SampleRowsArgs A{logits_dev, row_stride, vocab,       temperature_dev, top_p_dev,
                         min_p_dev,  uniform_dev, top_k_dev, tokens_dev,      probs_dev};
        if (dtype == FB_F32) k_sample_rows<float><<<(unsigned)rows, SR_THREADS, 0, ctx->stream>>>(A);
        else if (dtype == FB_F16) k_sample_rows<__half><<<(unsigned)rows, SR_THREADS, 0, ctx->stream>>>(A);
        else k_sample_rows<__nv_bfloat16><<<(unsigned)rows, SR_THREADS, 0, ctx->stream>>>(A);
        FB_CUDA(cudaGetLastError());
    });
}
