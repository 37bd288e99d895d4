// Rotary positions given per row, and the append of new rows to the paged
// cache (fb_rotary_*, fb_kv_append).  No reference counterpart: candle's RoPE
// (ptx-kernels/kernels/candle/reduce.cu:275-318) turns whole heads at
// consecutive positions and its cache grows by concatenation.
//
// Mathematics: pair i of a head turns by the angle a = pos * f_i,
//   (x0, x1) -> A (x0 cos a - x1 sin a, x0 sin a + x1 cos a).
// The frequencies are kept in turns a position (f_i / 2 pi) in binary64: the
// product pos * turns has an absolute error below 2^-53 of its size, its
// whole turns drop out exactly, and the remaining eighth of a turn at most is
// what sincospif sees, so a far position costs no precision.
//
// Bound: every value is read and written once, but memory is not what these
// kernels wait for (13 to 18 % of DRAM's rate from cold caches, 50 to 62 % of the
// issue slots).  A block of the rotation begins with binary64 angles and a barrier,
// and 2048 tokens are 1.7 waves of blocks; one token's call is a launch and two
// dependent loads; the append's transposing tiles are steps one after another.
// Measured (back to back in a graph, inputs warm in L2; in brackets from cold
// caches; 6559 GB/s the copy rate): 2048 tokens x 32 heads of 128, f16, 33.6 MB:
// 8.3 us (12.3); 777 x 64 heads with half a head turned, bf16, 25.5 MB: 8.0 us
// (12.4); one token 2.2 us (5.5).  The append: three prompts of up to 2731 bf16 rows
// of 8 heads, 56 MB: 14.5 us (18.7); 400 drafted rows 6.5 us (10.5).
#include <math.h>

#include <memory>

#include "fb_internal.h"
#include "kq_common.cuh"

struct fb_rotary {
    fb_rotary_config cfg;
    double freq[128];   // radians a position
    double amplitude;
};

namespace fb {

constexpr int ROT_MAX = 256;
constexpr int ROT_THREADS = 256;

// By value in the launch parameters (1 KB): a captured launch keeps its copy,
// and the handle needs no device memory.
struct RotaryParams {
    double turns[ROT_MAX / 2];  // turns a position
    float amp;
    int rot, mode;
};

static RotaryParams rotary_params(const fb_rotary *r) {
    RotaryParams p{};
    p.amp = 1.f;
    p.mode = 1;
    if (!r) return p;
    p.rot = r->cfg.rot_dim;
    p.mode = r->cfg.mode;
    p.amp = (float)r->amplitude;
    for (int i = 0; i < p.rot / 2; i++) p.turns[i] = r->freq[i] / (2.0 * M_PI);
    return p;
}

// A cos, A sin of pair i at position pos.  q = the nearest quarter turn: the
// rest is within an eighth of a turn, so its f32 rounding is below 2^-28 turns.
__device__ __forceinline__ float2 rotary_trig(const RotaryParams &p, int i, int pos) {
    const double t = (double)pos * p.turns[i];
    const double q = rint(4.0 * t);
    const float rest = (float)__fma_rn(q, -0.25, t);
    float s, c;
    sincospif(2.f * rest, &s, &c);
    const int quarter = (int)((long long)q & 3);
    float cc = (quarter & 1) ? -s : c, ss = (quarter & 1) ? c : s;
    if (quarter & 2) {
        cc = -cc;
        ss = -ss;
    }
    return make_float2(__fmul_rn(cc, p.amp), __fmul_rn(ss, p.amp));
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// One work unit: NP pairs of one head.  VEC: 16-byte accesses (mode 1: NP =
// 16 / sizeof(T) dimensions of either half; mode 0: half as many pairs of one
// vector); otherwise one pair, element by element.
template <typename T, bool VEC, int MODE> struct RotUnit {
    static constexpr int V = VEC ? 16 / (int)sizeof(T) : 1;
    static constexpr int NP = VEC ? (MODE == 1 ? V : V / 2) : 1;
    alignas(16) T a[VEC && MODE == 0 ? V : NP];
    alignas(16) T b[VEC && MODE == 0 ? 1 : NP];
    __device__ __forceinline__ void load(const T *x, int u, int rot) {
        if constexpr (VEC) {
            *reinterpret_cast<uint4 *>(a) = *reinterpret_cast<const uint4 *>(x + u * V);
            if constexpr (MODE == 1)
                *reinterpret_cast<uint4 *>(b) = *reinterpret_cast<const uint4 *>(x + rot / 2 + u * V);
        } else {
            a[0] = x[MODE == 1 ? u : 2 * u];
            b[0] = x[MODE == 1 ? u + rot / 2 : 2 * u + 1];
        }
    }
    __device__ __forceinline__ void turn(const float2 (&cs)[NP]) {
#pragma unroll
        for (int i = 0; i < NP; i++) {
            T &p0 = VEC && MODE == 0 ? a[2 * i] : a[i];
            T &p1 = VEC && MODE == 0 ? a[(2 * i + 1) % (VEC && MODE == 0 ? V : 1)] : b[i];
            const float x0 = to_f32(p0), x1 = to_f32(p1);
            p0 = from_f32<T>(__fsub_rn(__fmul_rn(x0, cs[i].x), __fmul_rn(x1, cs[i].y)));
            p1 = from_f32<T>(__fadd_rn(__fmul_rn(x0, cs[i].y), __fmul_rn(x1, cs[i].x)));
        }
    }
    __device__ __forceinline__ void store(T *y, int u, int rot) const {
        if constexpr (VEC) {
            *reinterpret_cast<uint4 *>(y + u * V) = *reinterpret_cast<const uint4 *>(a);
            if constexpr (MODE == 1)
                *reinterpret_cast<uint4 *>(y + rot / 2 + u * V) = *reinterpret_cast<const uint4 *>(b);
        } else {
            y[MODE == 1 ? u : 2 * u] = a[0];
            y[MODE == 1 ? u + rot / 2 : 2 * u + 1] = b[0];
        }
    }
};

// grid (tiles of tt tokens, shares of a tile's (token, head) items): thread = (item
// slot, unit of a head), unit fastest.  A unit is a rotated one or, behind those
// and unless the rotation is in place, a vector to copy.  A thread has the values
// of up to ROT_AHEAD items in flight while the tile's angles are computed, an
// angle a thread.
constexpr int ROT_AHEAD = 2;
template <typename T, bool VEC, int MODE>
__global__ void __launch_bounds__(ROT_THREADS)
    k_rotary(const __grid_constant__ RotaryParams P, const T *x, int64_t xt, int64_t xh, T *y, int64_t yt, int64_t yh,
             const int32_t *__restrict__ positions, int64_t n_tok, int n_heads, int dim, int tt, int items) {
    using U = RotUnit<T, VEC, MODE>;
    extern __shared__ float2 trig[];  // [tt][rot / 2]
    const int half = P.rot / 2, turned = half / U::NP;
    const bool copies = x != y && VEC;
    const int units = turned + (copies ? (dim - P.rot) / U::V : 0), slots = ROT_THREADS / units;
    const int64_t tok0 = (int64_t)blockIdx.x * tt;
    const int unit = threadIdx.x % units, slot = threadIdx.x / units;
    const int ntok = (int)min((int64_t)tt, n_tok - tok0);
    const int first = blockIdx.y * items, last = min(first + items, ntok * n_heads);
    const bool turn = unit < turned, active = slot < slots;
    const int rest0 = P.rot + (unit - turned) * U::V;  // of a copied vector
    U w[ROT_AHEAD];
    auto fetch = [&](int i0) {
#pragma unroll
        for (int k = 0; k < ROT_AHEAD; k++) {
            const int i = i0 + k * slots;
            if (!active || i >= last) continue;
            const int t = i / n_heads;
            const T *src = x + (tok0 + t) * xt + (i - t * n_heads) * xh;
            if (turn) w[k].load(src, unit, P.rot);
            else if constexpr (VEC) *reinterpret_cast<uint4 *>(w[k].a) = *reinterpret_cast<const uint4 *>(src + rest0);
        }
    };
    fetch(first + slot);
    for (int e = threadIdx.x; e < ntok * half; e += ROT_THREADS) {
        const int t = e / half;
        trig[e] = rotary_trig(P, e - t * half, positions[tok0 + t]);
    }
    __syncthreads();
    for (int i0 = first + slot; i0 < last; i0 += ROT_AHEAD * slots) {
        if (i0 != first + slot) fetch(i0);
#pragma unroll
        for (int k = 0; k < ROT_AHEAD; k++) {
            const int i = i0 + k * slots;
            if (!active || i >= last) break;
            const int t = i / n_heads;
            T *dst = y + (tok0 + t) * yt + (i - t * n_heads) * yh;
            if (turn) {
                float2 cs[U::NP];
#pragma unroll
                for (int j = 0; j < U::NP; j++) cs[j] = trig[t * half + unit * U::NP + j];
                w[k].turn(cs);
                w[k].store(dst, unit, P.rot);
            } else if constexpr (VEC) {
                *reinterpret_cast<uint4 *>(dst + rest0) = *reinterpret_cast<const uint4 *>(w[k].a);
            }
        }
    }
    if constexpr (!VEC) {  // element by element: the dimensions behind the rotated ones
        const int rest = dim - P.rot;
        if (x != y && rest > 0)
            for (int e = threadIdx.x; e < (last - first) * rest; e += ROT_THREADS) {
                const int d = P.rot + e % rest, i = first + e / rest, t = i / n_heads, h = i - t * n_heads;
                y[(tok0 + t) * yt + h * yh + d] = x[(tok0 + t) * xt + h * xh + d];
            }
    }
}

template <typename T, bool VEC, int MODE>
static void launch_rotary_as(fb_ctx *ctx, const RotaryParams &P, const T *x, int64_t xt, int64_t xh, T *y, int64_t yt,
                             int64_t yh, const int32_t *positions, int64_t n_tok, int n_heads, int dim) {
    using U = RotUnit<T, VEC, MODE>;
    const int units = P.rot / 2 / U::NP + (VEC && x != y ? (dim - P.rot) / U::V : 0);  // 1..256
    const int slots = ROT_THREADS / units;
    // tokens a block: as many as keep ROT_AHEAD items a thread in flight (and 2048 angles at most), fewer
    // while blocks are scarcer than two a SM; then a token's heads over several blocks
    int tt = (ROT_AHEAD * slots + n_heads - 1) / n_heads;
    if (tt > 4096 / P.rot) tt = 4096 / P.rot;
    while (tt > 1 && (n_tok + tt - 1) / tt < 2 * ctx->num_sms) tt = (tt + 1) / 2;
    const int64_t gx = (n_tok + tt - 1) / tt;
    FB_REQUIRE(gx <= 0x7fffffff, "rotary_apply: too many tokens");
    int64_t gy = (tt * (int64_t)n_heads + slots - 1) / slots;  // blocks with an item a thread
    if (gx * gy > ctx->num_sms) gy = gx >= ctx->num_sms ? 1 : ctx->num_sms / gx;
    const int items = (int)((tt * (int64_t)n_heads + gy - 1) / gy);
    const size_t smem = (size_t)tt * (P.rot / 2) * sizeof(float2);
    k_rotary<T, VEC, MODE><<<dim3((unsigned)gx, (unsigned)gy), ROT_THREADS, smem, ctx->stream>>>(
        P, x, xt, xh, y, yt, yh, positions, n_tok, n_heads, dim, tt, items);
    FB_CUDA(cudaGetLastError());
}

template <typename T>
static void launch_rotary(fb_ctx *ctx, const RotaryParams &P, const void *xv, int64_t xt, int64_t xh, void *yv,
                          int64_t yt, int64_t yh, const int32_t *positions, int64_t n_tok, int n_heads, int dim) {
    constexpr int V = 16 / (int)sizeof(T);
    const T *x = static_cast<const T *>(xv);
    T *y = static_cast<T *>(yv);
    // 16-byte accesses: every head starts on 16 bytes, the rotated part (its halves in mode 1) is whole vectors, and
    // a head is no more of them than a block has threads
    const bool vec = (((uintptr_t)xv | (uintptr_t)yv) & 15) == 0 && (xt | xh | yt | yh) % V == 0 && dim % V == 0 &&
                     (P.mode == 1 ? P.rot / 2 : P.rot) % V == 0 && dim / V <= ROT_THREADS;
    auto go = [&](auto v, auto m) {
        launch_rotary_as<T, decltype(v)::value, decltype(m)::value>(ctx, P, x, xt, xh, y, yt, yh, positions, n_tok,
                                                                    n_heads, dim);
    };
    using std::integral_constant;
    if (vec && P.mode == 1) go(integral_constant<bool, true>{}, integral_constant<int, 1>{});
    else if (vec) go(integral_constant<bool, true>{}, integral_constant<int, 0>{});
    else if (P.mode == 1) go(integral_constant<bool, false>{}, integral_constant<int, 1>{});
    else go(integral_constant<bool, false>{}, integral_constant<int, 0>{});
}

// ------------------------------------------------------------ cache append
constexpr int KVA_THREADS = 256;

struct AppendArgs {
    const void *k, *v;
    int64_t kt, vt;
    const int32_t *offsets, *lens, *positions, *bt;
    __half *kpool, *vpool;
    int n_rows, max_new, n_kv, page, max_pages, num_pages, heads_per_block;
    bool vec;  // k and v rows start on 16 bytes
    uint32_t *err;
};

// Eight consecutive values of a row as f32.
template <typename T> __device__ __forceinline__ void load8(const T *p, bool vec, float (&v)[8]) {
    alignas(16) T t[8];
    if (vec) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++)
            reinterpret_cast<uint4 *>(t)[i] = reinterpret_cast<const uint4 *>(p)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) t[i] = p[i];
    }
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = to_f32(t[i]);
}
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t *>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// The part of a sequence's new rows that falls into this block's page: cache
// positions from .. to - 1, the page's id, the first row.  False: nothing to do.
__device__ __forceinline__ bool append_span(const AppendArgs &A, int &from, int &to, int &phys, int &row0) {
    const int b = blockIdx.z;
    const int off = A.offsets[b], n = A.offsets[b + 1] - off, len = A.lens[b];
    if (off < 0 || n < 0 || n > A.max_new || off > A.n_rows - n || len < n || len > A.max_pages * A.page) {
        if (threadIdx.x == 0) atomicOr(A.err, ERRBIT_BAD_POS);
        return false;
    }
    const int p0 = len - n, pg = p0 / A.page + blockIdx.x;
    from = max(p0, pg * A.page);
    to = min(len, (pg + 1) * A.page);
    if (from >= to) return false;
    phys = A.bt[(int64_t)b * A.max_pages + pg];
    if (phys < 0 || phys >= A.num_pages) {
        if (threadIdx.x == 0) atomicOr(A.err, ERRBIT_BAD_PAGE);
        return false;
    }
    row0 = off + from - p0;
    return true;
}

// Eight values of a row as they are stored.
template <typename T> struct Raw8 {
    uint4 q[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T *p) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) q[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = to_f32(reinterpret_cast<const T *>(q)[i]);
    }
};

// grid (pages a sequence's new rows can touch, kv head groups, batch): a block
// writes the new rows that fall into one page, for up to KVA_HEADS heads.  A warp
// takes 8 rows x 4 units (8 dimensions, in mode 1 with the 8 they are paired
// with): the angles of a unit are computed once and serve all heads; the rotated
// keys go as fp16 into a [dim][token] tile whose 16-byte token chunks are
// exchanged by the dimension's chunk (both the scattered 2-byte stores and the
// rows' 16-byte loads then touch every bank once).  The pages are dim-major: 8
// lanes write the 128 bytes of a dimension's 64 tokens.
constexpr int KVA_HEADS = 2;  // (three prompts: 14.3 us; 15.3 with 4, 16.0 with 1)
template <typename T, int HD, int PAGE, int MODE>
__global__ void __launch_bounds__(KVA_THREADS)
    k_kv_append(const __grid_constant__ RotaryParams P, const __grid_constant__ AppendArgs A) {
    extern __shared__ __align__(16) uint8_t kva_tile[];  // [head][HD][PAGE] fp16
    constexpr int CH = PAGE / 8;
    int from, to, phys, row0;
    if (!append_span(A, from, to, phys, row0)) return;
    const int cnt = to - from, t0 = from % PAGE;
    const int h0 = blockIdx.y * A.heads_per_block, nh = min(A.heads_per_block, A.n_kv - h0);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const T *kr = static_cast<const T *>(A.k) + (int64_t)row0 * A.kt + (int64_t)h0 * HD;
    const T *vr = static_cast<const T *>(A.v) + (int64_t)row0 * A.vt + (int64_t)h0 * HD;
    __half *kp = A.kpool + ((int64_t)phys * A.n_kv + h0) * HD * PAGE;
    __half *vp = A.vpool + ((int64_t)phys * A.n_kv + h0) * HD * PAGE + (int64_t)t0 * HD;
    const int half = P.rot / 2;
    // units of a row: mode 1 rot / 16 pairs of chunks and the chunks behind them, mode 0 all chunks
    const int paired = MODE == 1 ? P.rot / 16 : 0, nu = paired + (MODE == 1 ? (HD - P.rot) / 8 : HD / 8);
    const int ug = (nu + 3) / 4, tg = (cnt + 7) / 8;
    auto put = [&](int h, int c, int t, const float (&v)[8]) {  // chunk c of head h, token t of the page
        __half *tile = reinterpret_cast<__half *>(kva_tile) + h * HD * PAGE;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int d = 8 * c + i;
            tile[d * PAGE + (((t >> 3) ^ (c & (CH - 1))) << 3) + (t & 7)] = __float2half_rn(v[i]);
        }
    };
    // V rows, as they come (first: K waits for its angles anyway)
    for (int e = threadIdx.x; e < cnt * nh * (HD / 8); e += KVA_THREADS) {
        const int c = e % (HD / 8), q = e / (HD / 8), h = q % nh, t = q / nh;
        Raw8<T> raw;
        raw.load(vr + t * A.vt + h * HD + 8 * c);
        float v[8];
        raw.get(v);
        *reinterpret_cast<uint4 *>(vp + (int64_t)h * HD * PAGE + t * HD + 8 * c) = pack8(v);
    }
    for (int wt = warp; wt < ug * tg; wt += KVA_THREADS / 32) {
        const int u = (wt % ug) * 4 + (lane & 3), t = (wt / ug) * 8 + (lane >> 2);
        if (u >= nu || t >= cnt) continue;
        const bool pair = u < paired;
        const int c = MODE == 1 ? (pair ? u : 2 * paired + (u - paired)) : u;  // the unit's (first) chunk
        const int c2 = c + (MODE == 1 ? half / 8 : 0);
        const bool turn = MODE == 1 ? pair : 8 * c < P.rot;
        const T *src = kr + t * A.kt;
        constexpr int AH = 2;  // heads in flight
        Raw8<T> a[AH], b[AH];
        auto fetch = [&](int h) {
#pragma unroll
            for (int k = 0; k < AH; k++)
                if (h + k < nh) {
                    a[k].load(src + (h + k) * HD + 8 * c);
                    if (MODE == 1 && pair) b[k].load(src + (h + k) * HD + 8 * c2);
                }
        };
        fetch(0);
        constexpr int NP = MODE == 1 ? 8 : 4;
        float2 cs[NP];
        if (turn) {
            const int pos = A.positions ? A.positions[row0 + t] : from + t;
#pragma unroll
            for (int i = 0; i < NP; i++) cs[i] = rotary_trig(P, MODE == 1 ? 8 * c + i : 4 * c + i, pos);
        }
        for (int h = 0; h < nh; h += AH) {
            if (h > 0) fetch(h);
#pragma unroll
            for (int k = 0; k < AH; k++) {
                if (h + k >= nh) break;
                float x[8], y[8];
                a[k].get(x);
                if (MODE == 1 && pair) b[k].get(y);
                if (turn) {
#pragma unroll
                    for (int i = 0; i < NP; i++) {
                        float &p0 = MODE == 1 ? x[i] : x[(2 * i) & 7], &p1 = MODE == 1 ? y[i] : x[(2 * i + 1) & 7];
                        const float x0 = p0, x1 = p1;
                        p0 = __fsub_rn(__fmul_rn(x0, cs[i].x), __fmul_rn(x1, cs[i].y));
                        p1 = __fadd_rn(__fmul_rn(x0, cs[i].y), __fmul_rn(x1, cs[i].x));
                    }
                }
                put(h + k, c, t0 + t, x);
                if (MODE == 1 && pair) put(h + k, c2, t0 + t, y);
            }
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < nh * HD * CH; e += KVA_THREADS) {
        const int c = e % CH, d = e / CH;  // (heads follow one another in the tile and in the page)
        if (8 * c + 8 <= t0 || 8 * c >= t0 + cnt) continue;
        const __half *src = reinterpret_cast<const __half *>(kva_tile) + d * PAGE + ((c ^ ((d >> 3) & (CH - 1))) << 3);
        __half *dst = kp + (int64_t)d * PAGE + 8 * c;
        if (8 * c >= t0 && 8 * c + 8 <= t0 + cnt) {
            *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(src);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (8 * c + j >= t0 && 8 * c + j < t0 + cnt) dst[j] = src[j];
        }
    }
}

// The general form: any rot_dim, any alignment.  K is staged as f32 rows in shared
// memory and rotated on its way out.
template <typename T, int HD>
__global__ void __launch_bounds__(KVA_THREADS)
    k_kv_append_any(const __grid_constant__ RotaryParams P, const __grid_constant__ AppendArgs A) {
    extern __shared__ float kva_smem[];
    constexpr int PITCH = HD + 1;
    float *rows = kva_smem;                                             // [page][PITCH]
    float2 *trig = reinterpret_cast<float2 *>(kva_smem + A.page * PITCH + (A.page * PITCH & 1));  // [page][half + 1]
    int from, to, phys, row0;
    if (!append_span(A, from, to, phys, row0)) return;
    const int cnt = to - from, t0 = from % A.page;
    const int half = P.rot / 2;
    for (int e = threadIdx.x; e < cnt * half; e += KVA_THREADS) {
        const int t = e / half, i = e - t * half;
        trig[t * (half + 1) + i] = rotary_trig(P, i, A.positions ? A.positions[row0 + t] : from + t);
    }
    const int h_end = min(A.n_kv, (int)(blockIdx.y + 1) * A.heads_per_block);
    for (int h = blockIdx.y * A.heads_per_block; h < h_end; h++) {
        const T *ksrc = static_cast<const T *>(A.k) + (int64_t)row0 * A.kt + (int64_t)h * HD;
        const T *vsrc = static_cast<const T *>(A.v) + (int64_t)row0 * A.vt + (int64_t)h * HD;
        __half *kdst = A.kpool + ((int64_t)phys * A.n_kv + h) * HD * A.page;
        __half *vdst = A.vpool + ((int64_t)phys * A.n_kv + h) * HD * A.page + (int64_t)t0 * HD;
        __syncthreads();  // the previous head's rows have been read
        for (int e = threadIdx.x; e < cnt * (HD / 8); e += KVA_THREADS) {
            const int t = e / (HD / 8), c = e % (HD / 8);
            float kx[8], vx[8];
            load8(ksrc + t * A.kt + c * 8, A.vec, kx);
            load8(vsrc + t * A.vt + c * 8, A.vec, vx);
#pragma unroll
            for (int i = 0; i < 8; i++) rows[t * PITCH + c * 8 + i] = kx[i];
            *reinterpret_cast<uint4 *>(vdst + t * HD + c * 8) = pack8(vx);
        }
        __syncthreads();
        const int chunks = A.page / 8;
        for (int e = threadIdx.x; e < HD * chunks; e += KVA_THREADS) {
            const int d = e / chunks, c = e % chunks;  // dimension, tokens 8 c .. 8 c + 7 of the page
            if (8 * c + 8 <= t0 || 8 * c >= t0 + cnt) continue;
            // the pair of dimension d: its partner's distance, and its angle's index
            int other = 0, i = 0;
            float sign = 0.f;
            if (d < P.rot) {
                const bool first = P.mode == 1 ? d < half : (d & 1) == 0;
                i = P.mode == 1 ? (first ? d : d - half) : d >> 1;
                other = P.mode == 1 ? (first ? half : -half) : (first ? 1 : -1);
                sign = first ? -1.f : 1.f;
            }
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int t = 8 * c + j - t0;
                v[j] = 0.f;
                if (t < 0 || t >= cnt) continue;
                v[j] = rows[t * PITCH + d];
                if (d < P.rot) {
                    const float2 cs = trig[t * (half + 1) + i];
                    v[j] = __fadd_rn(__fmul_rn(v[j], cs.x), __fmul_rn(sign * cs.y, rows[t * PITCH + d + other]));
                }
            }
            __half *dst = kdst + (int64_t)d * A.page + 8 * c;
            if (8 * c >= t0 && 8 * c + 8 <= t0 + cnt) {
                *reinterpret_cast<uint4 *>(dst) = pack8(v);
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (8 * c + j >= t0 && 8 * c + j < t0 + cnt) dst[j] = __float2half_rn(v[j]);
            }
        }
    }
}

// Shared memory of the general form: f32 rows and angles.
constexpr size_t append_any_bytes(int page, int hd, int rot) {
    return (size_t)(page * (hd + 1) + 1) * 4 + (size_t)page * (rot / 2 + 1) * 8;
}

template <typename T, int HD, int PAGE>
static void launch_append(fb_ctx *ctx, const RotaryParams &P, AppendArgs A, int batch) {
    const int tiles = (A.max_new + PAGE - 2) / PAGE + 1;
    // heads of a block share its angles; with fewer than two blocks a SM each has a block of its own
    const int64_t blocks = (int64_t)tiles * batch * A.n_kv;
    const int64_t hpb = blocks / (2 * ctx->num_sms);
    A.heads_per_block = hpb < 1 ? 1 : hpb > A.n_kv ? A.n_kv : (int)hpb;
    // 16-byte loads and whole chunks of 8 dimensions (of either half in mode 1)
    const bool fast = A.vec && P.rot % (P.mode == 1 ? 16 : 8) == 0;
    if (fast && A.heads_per_block > KVA_HEADS) A.heads_per_block = KVA_HEADS;
    const dim3 grid((unsigned)tiles, (unsigned)((A.n_kv + A.heads_per_block - 1) / A.heads_per_block), (unsigned)batch);
    // most: the kernel's bound for its shared-memory limit, not this call's size: the limit belongs to the process, whose
    // other threads launch other sizes
    auto go = [&](auto kernel, size_t smem, size_t most) {
        FB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
        kernel<<<grid, KVA_THREADS, smem, ctx->stream>>>(P, A);
        FB_CUDA(cudaGetLastError());
    };
    const size_t tile = (size_t)A.heads_per_block * HD * PAGE * 2;
    constexpr size_t tiles_most = (size_t)KVA_HEADS * HD * PAGE * 2;
    if (!fast) go(k_kv_append_any<T, HD>, append_any_bytes(PAGE, HD, P.rot), append_any_bytes(64, HD, HD));
    else if (P.mode == 1) go(k_kv_append<T, HD, PAGE, 1>, tile, tiles_most);
    else go(k_kv_append<T, HD, PAGE, 0>, tile, tiles_most);
}

}  // namespace fb

using namespace fb;

extern "C" {

int fb_rotary_create(const fb_rotary_config *cfg, fb_rotary **out) {
    return guarded([&] {
        FB_REQUIRE(cfg && out, "null argument");
        *out = nullptr;
        fb_rotary_config c = *cfg;
        FB_REQUIRE(c.rot_dim >= 2 && c.rot_dim <= ROT_MAX && c.rot_dim % 2 == 0,
                   "rotary: rot_dim must be even, 2..256");
        FB_REQUIRE(c.mode == 0 || c.mode == 1, "rotary: mode must be 0 or 1");
        FB_REQUIRE(c.scaling >= FB_ROTARY_PLAIN && c.scaling <= FB_ROTARY_YARN, "rotary: unknown scaling");
        FB_REQUIRE(isfinite(c.theta) && c.theta > 1.0, "rotary: theta must be above 1");
        FB_REQUIRE(isfinite(c.amplitude) && c.amplitude >= 0.0, "rotary: amplitude must not be negative");
        if (c.scaling != FB_ROTARY_PLAIN)
            FB_REQUIRE(isfinite(c.factor) && c.factor >= 1e-6, "rotary: factor must be positive, 1e-6 at least");
        if (c.scaling == FB_ROTARY_BANDS || c.scaling == FB_ROTARY_YARN) {
            FB_REQUIRE(c.orig_ctx >= 1, "rotary: orig_ctx must be positive");
            FB_REQUIRE(isfinite(c.high) && c.low > 0.0 && c.high > c.low, "rotary: need 0 < low < high");
        }
        auto r = std::make_unique<fb_rotary>();
        r->cfg = c;
        r->amplitude = c.amplitude > 0.0 ? c.amplitude : c.scaling == FB_ROTARY_YARN ? 0.1 * log(c.factor) + 1.0 : 1.0;
        FB_REQUIRE(r->amplitude > 0.0, "rotary: YaRN's own amplitude is not positive at this factor: give one");
        const double ctx_len = (double)c.orig_ctx;
        double a = 0.0, b = 0.0;
        if (c.scaling == FB_ROTARY_YARN) {
            // the (fractional) pair index that makes `turns` turns over the original context
            auto index_of = [&](double turns) {
                return c.rot_dim * log(ctx_len / (2.0 * M_PI * turns)) / (2.0 * log(c.theta));
            };
            a = fmax(floor(index_of(c.high)), 0.0);
            b = fmin(ceil(index_of(c.low)), (double)(c.rot_dim - 1));
        }
        for (int i = 0; i < c.rot_dim / 2; i++) {
            const double f = pow(c.theta, -2.0 * i / c.rot_dim);
            double g = 0.0;  // share of the interpolated frequency f / factor
            if (c.scaling == FB_ROTARY_LINEAR) g = 1.0;
            else if (c.scaling == FB_ROTARY_BANDS)
                g = 1.0 - fmin(fmax((ctx_len * f / (2.0 * M_PI) - c.low) / (c.high - c.low), 0.0), 1.0);
            else if (c.scaling == FB_ROTARY_YARN) g = fmin(fmax((i - a) / fmax(b - a, 0.001), 0.0), 1.0);
            r->freq[i] = g == 0.0 ? f : f * (1.0 - g) + f / c.factor * g;
        }
        *out = r.release();
    });
}

int fb_rotary_destroy(fb_rotary *r) {
    return guarded([&] { delete r; });
}

int fb_rotary_frequencies(const fb_rotary *r, double *freq_host, int capacity, double *amplitude) {
    return guarded([&] {
        FB_REQUIRE(r && freq_host, "null argument");
        FB_REQUIRE(capacity >= r->cfg.rot_dim / 2, "rotary_frequencies: capacity must be at least rot_dim / 2");
        for (int i = 0; i < r->cfg.rot_dim / 2; i++) freq_host[i] = r->freq[i];
        if (amplitude) *amplitude = r->amplitude;
    });
}

int fb_rotary_apply(fb_ctx *ctx, const fb_rotary *r, int dtype, const void *x_dev, int64_t x_token_stride,
                    int64_t x_head_stride, void *y_dev, int64_t y_token_stride, int64_t y_head_stride,
                    const int32_t *positions_dev, int64_t n_tok, int n_heads, int head_dim) {
    return guarded([&] {
        FB_REQUIRE(r, "rotary_apply: null rotary handle");
        FB_REQUIRE(dtype == FB_F32 || dtype == FB_F16 || dtype == FB_BF16,
                   "rotary_apply: dtype must be FB_F32, FB_F16 or FB_BF16");
        FB_REQUIRE(n_tok >= 0 && n_heads >= 1 && n_heads <= 65535 && head_dim >= 1 && head_dim <= 1024,
                   "rotary_apply: bad shape");
        FB_REQUIRE(r->cfg.rot_dim <= head_dim, "rotary_apply: rot_dim exceeds head_dim");
        FB_REQUIRE(x_token_stride >= 0 && x_head_stride >= 0 && y_token_stride >= 0 && y_head_stride >= 0,
                   "rotary_apply: strides must not be negative");
        // one stride steps over all that the other spans
        FB_REQUIRE((n_heads == 1 || y_head_stride >= head_dim) && (n_tok <= 1 || y_token_stride >= head_dim) &&
                       (n_heads == 1 || n_tok <= 1 || (y_token_stride - head_dim) / (n_heads - 1) >= y_head_stride ||
                        (y_head_stride - head_dim) / (n_tok - 1) >= y_token_stride),
                   "rotary_apply: rows of y overlap");
        FB_REQUIRE(x_dev != y_dev || (x_token_stride == y_token_stride && x_head_stride == y_head_stride),
                   "rotary_apply: in place needs equal strides");
        if (n_tok == 0) return;
        FB_REQUIRE(ctx && x_dev && y_dev && positions_dev, "null argument");
        const size_t esz = dtype == FB_F32 ? 4 : 2;
        FB_REQUIRE((((uintptr_t)x_dev | (uintptr_t)y_dev) & (esz - 1)) == 0 && ((uintptr_t)positions_dev & 3) == 0,
                   "rotary_apply: misaligned pointer");
        FB_REQUIRE(x_dev == y_dev || !rows_overlap(x_dev, x_token_stride, x_head_stride, y_dev, y_token_stride,
                                                   y_head_stride, n_tok, n_heads, head_dim, esz),
                   "rotary_apply: x and y overlap");
        DeviceGuard guard(ctx->device);
        const RotaryParams P = rotary_params(r);
        switch (dtype) {
        case FB_F32:
            launch_rotary<float>(ctx, P, x_dev, x_token_stride, x_head_stride, y_dev, y_token_stride, y_head_stride,
                                 positions_dev, n_tok, n_heads, head_dim);
            break;
        case FB_F16:
            launch_rotary<__half>(ctx, P, x_dev, x_token_stride, x_head_stride, y_dev, y_token_stride, y_head_stride,
                                  positions_dev, n_tok, n_heads, head_dim);
            break;
        default:
            launch_rotary<__nv_bfloat16>(ctx, P, x_dev, x_token_stride, x_head_stride, y_dev, y_token_stride,
                                         y_head_stride, positions_dev, n_tok, n_heads, head_dim);
        }
    });
}

int fb_kv_append(fb_ctx *ctx, const fb_rotary *r, int dtype, const void *k_dev, int64_t k_token_stride,
                 const void *v_dev, int64_t v_token_stride, const int32_t *row_offsets_dev,
                 const int32_t *seq_lens_dev, const int32_t *positions_dev, const int32_t *block_table_dev,
                 void *k_pages_dev, void *v_pages_dev, int batch, int n_rows, int max_new, int n_kv_heads,
                 int head_dim, int page_size, int max_pages, int num_pages) {
    return guarded([&] {
        FB_REQUIRE(dtype == FB_F32 || dtype == FB_F16 || dtype == FB_BF16,
                   "kv_append: dtype must be FB_F32, FB_F16 or FB_BF16");
        FB_REQUIRE(head_dim == 64 || head_dim == 128, "kv_append: head_dim must be 64 or 128");
        FB_REQUIRE(page_size == 32 || page_size == 64, "kv_append: page_size must be 32 or 64");
        FB_REQUIRE(batch >= 0 && batch <= 65535 && n_rows >= 0 && max_new >= 0 && n_kv_heads >= 1 &&
                       n_kv_heads <= 65535 && max_pages >= 1 && num_pages >= 1,
                   "kv_append: bad shape");
        FB_REQUIRE((int64_t)max_pages * page_size <= ((int64_t)1 << 30), "kv_append: block table too long");
        FB_REQUIRE(max_new <= max_pages * page_size, "kv_append: max_new exceeds the block table");
        FB_REQUIRE(!r || r->cfg.rot_dim <= head_dim, "kv_append: rot_dim exceeds head_dim");
        FB_REQUIRE(k_token_stride >= 0 && v_token_stride >= 0, "kv_append: strides must not be negative");
        if (batch == 0 || n_rows == 0 || max_new == 0) return;
        FB_REQUIRE(ctx && k_dev && v_dev && row_offsets_dev && seq_lens_dev && block_table_dev && k_pages_dev &&
                       v_pages_dev,
                   "null argument");
        const size_t esz = dtype == FB_F32 ? 4 : 2;
        FB_REQUIRE((((uintptr_t)k_dev | (uintptr_t)v_dev) & (esz - 1)) == 0 &&
                       (((uintptr_t)row_offsets_dev | (uintptr_t)seq_lens_dev | (uintptr_t)block_table_dev |
                         (uintptr_t)positions_dev) & 3) == 0,
                   "kv_append: misaligned pointer");
        FB_REQUIRE((((uintptr_t)k_pages_dev | (uintptr_t)v_pages_dev) & 15) == 0,
                   "kv_append: KV pools must be 16-byte aligned");
        DeviceGuard guard(ctx->device);
        const int V = (int)(16 / esz);
        AppendArgs A{};
        A.k = k_dev;
        A.v = v_dev;
        A.kt = k_token_stride;
        A.vt = v_token_stride;
        A.offsets = row_offsets_dev;
        A.lens = seq_lens_dev;
        A.positions = positions_dev;
        A.bt = block_table_dev;
        A.kpool = static_cast<__half *>(k_pages_dev);
        A.vpool = static_cast<__half *>(v_pages_dev);
        A.n_rows = n_rows;
        A.max_new = max_new;
        A.n_kv = n_kv_heads;
        A.page = page_size;
        A.max_pages = max_pages;
        A.num_pages = num_pages;
        A.vec = (((uintptr_t)k_dev | (uintptr_t)v_dev) & 15) == 0 && (k_token_stride | v_token_stride) % V == 0;
        A.err = ctx->err_word;
        const RotaryParams P = rotary_params(r);
        auto go = [&](auto t) {
            using T = decltype(t);
            if (head_dim == 128 && page_size == 64) launch_append<T, 128, 64>(ctx, P, A, batch);
            else if (head_dim == 128) launch_append<T, 128, 32>(ctx, P, A, batch);
            else if (page_size == 64) launch_append<T, 64, 64>(ctx, P, A, batch);
            else launch_append<T, 64, 32>(ctx, P, A, batch);
        };
        if (dtype == FB_F32) go(float{});
        else if (dtype == FB_F16) go(__half{});
        else go(__nv_bfloat16{});
    });
}

}  // extern "C"
