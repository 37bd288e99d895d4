// Attention of drafted token trees over the paged cache (fb_attn_tree).  No
// reference counterpart: the reference verifies one chain, token by token
// (crates/ferrite-core/src/generation.rs:340-535).
//
// o = sum_j p_j v_j / sum_j p_j, p_j = exp(scale q.k_j - m), j over the prefix
// and the drafted tokens whose mask bit is set.
//
// The (drafted token, query head of the group) pairs of a sequence and kv head
// are the rows of one matrix product: 128 rows a tile share every key and
// value that is read.  A verified tree of 32 tokens with 4 heads a group needs
// 128 multiplications a byte of cache, so up to one full tile the bound is HBM
// (4 head_dim bytes a key and kv head), beyond it the tensor cores.
//
// Split: the (sequence, kv head, tile, 64-key block) units of a call are
// counted on the device from the lengths and dealt to one CTA per SM in equal
// contiguous shares, so unequal lengths and few sequences fill the machine
// alike.  A (sequence, kv head, tile) group that one CTA holds whole is written
// directly; the others leave (max, sum, o) partials, at most two a CTA, that a
// second kernel joins in share order (no atomics: the same bits every time).
// Calls of at most TR_WHOLE blocks a group deal whole groups and need no join.
//
// A CTA, 11 warps: 0..7 softmax (warp w: rows 32 (w % 4) .. + 31, keys 32 (w /
// 4) .. + 31 of a block), 8 and 10 TMA copies of K and V pages, 9 issues
// tcgen05.mma and owns the tensor memory.  The dim-major K pages and
// token-major V pages land in shared memory as the MN-major operands of S = Q
// K^T and O += P V.  S has two buffers, so the product of block j + 1 runs
// under the softmax of block j.  The roles run on through the CTA's groups: the
// next group's keys load and its queries are laid out while a group drains.
//
// Precision: q is scaled by a power of two a row (to 2^13..2^14 at most) and
// enters as fp16 high + low parts where it is f32 (f16 and bf16 queries fit
// the high part); the probabilities are kept 2^7 above the running maximum's
// unit (at most 2^15), so that high + low fp16 parts hold 22 bits down to 2^-21
// of the largest; products and sums are f32.  The accumulator is rescaled only
// when a row's maximum grows by more than 8 (log 2 units).
#include <math.h>

#include "fb_internal.h"
#include "kq_common.cuh"
#include "tc_common.cuh"

namespace fb {

struct TreeArgs {
    const void *q;
    int64_t qt, ot;
    const __half *kpool, *vpool;
    const int32_t *bt, *offsets, *lens;
    const uint32_t *mask;
    int mask_words;
    void *out;
    int batch, n_rows, max_new, n_heads, n_kv, max_pages, num_pages, max_seq;
    int group;      // query heads a kv head
    int split;      // 1: units are key blocks, 0: whole groups
    int ctas;       // CTAs of the attention kernel
    int rows_cap;   // row capacity of a partial (multiple of 32, <= 128)
    float *part;    // [2 ctas] partials of (head_dim + 2) rows_cap floats
    float scale;
    bool qvec, ovec;  // q / out rows start on 16 bytes
    uint32_t *err;
};

constexpr int TR_ROWS = 128;      // rows a tile (MMA M)
constexpr int TR_KB = 64;         // keys a block
constexpr int TR_WHOLE = 2;
constexpr int TR_THREADS = 352;
constexpr float TR_NONE = -1e30f;  // running maximum of a row that has seen nothing
constexpr float TR_LIFT = 7.f;     // probabilities are kept 2^7 above the reference maximum

__device__ __forceinline__ float tr_f32(float v) { return v; }
__device__ __forceinline__ float tr_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float tr_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void tr_put(float *p, float v) { *p = v; }
__device__ __forceinline__ void tr_put(__half *p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void tr_put(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

// Eight consecutive values of a row.
template <typename T> __device__ __forceinline__ void tr_load8(const T *p, bool vec, float (&v)[8]) {
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
    for (int i = 0; i < 8; i++) v[i] = tr_f32(t[i]);
}
template <typename T> __device__ __forceinline__ void tr_store8(T *p, bool vec, const float (&v)[8]) {
    alignas(16) T t[8];
#pragma unroll
    for (int i = 0; i < 8; i++) tr_put(t + i, v[i]);
    if (vec) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++)
            reinterpret_cast<uint4 *>(p)[i] = reinterpret_cast<const uint4 *>(t)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) p[i] = t[i];
    }
}

// One sequence of the batch: its new rows, key blocks, row tiles and groups
// (kv head major, tile minor).  A sequence left out has no groups.
struct TreeSeq {
    int off, n, len, blocks, tiles, groups;
    __device__ __forceinline__ bool load(const TreeArgs &A, int b) {
        off = A.offsets[b];
        n = A.offsets[b + 1] - off;
        len = A.lens[b];
        const bool ok = off >= 0 && n >= 0 && n <= A.max_new && off <= A.n_rows - n && len >= n && len <= A.max_seq;
        if (!ok) n = len = 0;
        blocks = (len + TR_KB - 1) / TR_KB;
        tiles = (n * A.group + TR_ROWS - 1) / TR_ROWS;
        groups = tiles * A.n_kv;
        return ok;
    }
    __device__ __forceinline__ int per_group(const TreeArgs &A) const { return A.split ? blocks : 1; }
    __device__ __forceinline__ int units(const TreeArgs &A) const { return groups * per_group(A); }
};

// Units of the whole call (every lane of the warp gets the sum).
__device__ __forceinline__ int tree_total(const TreeArgs &A, int lane, bool report) {
    int total = 0;
    for (int b = lane; b < A.batch; b += 32) {
        TreeSeq s;
        if (!s.load(A, b) && report) atomicOr(A.err, ERRBIT_BAD_POS);
        total += s.units(A);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    return total;
}
// A CTA's share; the join kernel derives the same one.
__device__ __forceinline__ int tree_quota(const TreeArgs &A, int total) { return (total + A.ctas - 1) / A.ctas; }

// The segments of a CTA's share [u0, u1): consecutive blocks of one group.
struct TreeWalk {
    TreeSeq s;
    int b, g, blk0, blk1, left;
    // warp-collective; u0 < u1 <= total
    __device__ __forceinline__ void start(const TreeArgs &A, int u0, int u1, int lane) {
        int base = 0;
        b = 0;
        for (int b0 = 0; b0 < A.batch; b0 += 32) {
            int mine = 0;
            if (b0 + lane < A.batch) {
                s.load(A, b0 + lane);
                mine = s.units(A);
            }
            int incl = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += y;
            }
            const uint32_t past = __ballot_sync(0xffffffffu, base + incl > u0);
            if (past) {
                const int w = __ffs(past) - 1;
                b = b0 + w;
                base += __shfl_sync(0xffffffffu, incl - mine, w);
                break;
            }
            base += __shfl_sync(0xffffffffu, incl, 31);
        }
        s.load(A, b);
        const int per = s.per_group(A), r = u0 - base;
        g = r / per;
        left = u1 - u0;
        span(A, r % per);
    }
    __device__ __forceinline__ void span(const TreeArgs &A, int first) {
        blk0 = A.split ? first : 0;
        blk1 = A.split ? min(s.blocks, blk0 + left) : s.blocks;
        left -= A.split ? blk1 - blk0 : 1;
    }
    __device__ __forceinline__ bool next(const TreeArgs &A) {
        if (left <= 0) return false;
        if (++g == s.groups) {
            g = 0;
            do {
                if (++b >= A.batch) return false;
                s.load(A, b);
            } while (s.units(A) == 0);
        }
        span(A, 0);
        return true;
    }
    __device__ __forceinline__ int head() const { return g / s.tiles; }
    __device__ __forceinline__ int row0() const { return (g % s.tiles) * TR_ROWS; }
    __device__ __forceinline__ int rows(const TreeArgs &A) const { return min(TR_ROWS, s.n * A.group - row0()); }
    __device__ __forceinline__ bool whole() const { return blk0 == 0 && blk1 == s.blocks; }
};

// Which of the keys p0 .. p0 + 31 new row i of a sequence sees.
__device__ __forceinline__ uint32_t tree_visible(const TreeArgs &A, const TreeSeq &s, int i, int p0) {
    const int pre = s.len - s.n, j0 = p0 - pre;  // first key's index among the new rows
    if (j0 <= -32) return 0xffffffffu;
    uint32_t v;
    if (A.mask) {
        const uint32_t *w = A.mask + (int64_t)(s.off + i) * A.mask_words;
        if (j0 < 0) {
            v = (w[0] << -j0) | ((1u << -j0) - 1u);
        } else {
            const int k = j0 >> 5, sh = j0 & 31;
            v = k < A.mask_words ? w[k] >> sh : 0u;
            if (sh && k + 1 < A.mask_words) v |= w[k + 1] << (32 - sh);
        }
    } else {
        const int last = i - j0;  // keys up to the row's own
        v = last < 0 ? 0u : last >= 31 ? 0xffffffffu : (2u << last) - 1u;
    }
    const int end = s.len - p0;
    return end <= 0 ? 0u : end >= 32 ? v : v & ((1u << end) - 1u);
}

template <typename T, int HD> struct TreeCfg {
    static constexpr bool QLO = sizeof(T) == 4;  // f32 queries need a low part
    static constexpr int ST = HD == 128 && QLO ? 3 : 4;  // K and V stages
    static constexpr uint32_t Q_BYTES = TR_ROWS * HD * 2;
    static constexpr uint32_t KV_BYTES = TR_KB * HD * 2;  // one block of K or V
    static constexpr uint32_t P_BYTES = TR_ROWS * TR_KB * 2;
    static constexpr size_t SMEM = 1024 + (QLO ? 2 : 1) * (size_t)Q_BYTES + 2 * ST * (size_t)KV_BYTES + 4 * (size_t)P_BYTES;
    static_assert(SMEM + 2048 <= 227 * 1024, "tree attention stages must fit");
};
constexpr uint32_t TR_TMEM_COLS = 256;  // S buffers at columns 0 and 64, O at 128
constexpr uint32_t TR_O_COL = 128;

template <typename T, int HD, int PAGE>
__global__ void __launch_bounds__(TR_THREADS, 1)
    k_attn_tree(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                const __grid_constant__ TreeArgs A) {
    using C = TreeCfg<T, HD>;
    constexpr int ST = C::ST, PPB = TR_KB / PAGE;  // pages a block
    constexpr uint32_t IDESC_S = umma_idesc_f16(TR_ROWS, TR_KB, false, true);
    constexpr uint32_t IDESC_O = umma_idesc_f16(TR_ROWS, HD, false, true);
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t k_full[ST], k_empty[ST], v_full[ST], v_empty[ST], s_full[2], s_free[2], p_full[2], p_free[2],
        q_full, o_free, fin, pair_bar[4];
    __shared__ uint32_t s_tmem;
    __shared__ float s_l[2][TR_ROWS];
    __shared__ uint8_t s_qe[2][TR_ROWS];  // exponent field of a row half's largest query value
    __shared__ int s_abort_raw, s_odd_raw[2];
    __shared__ uint8_t s_skip_raw[8];
    volatile int &s_abort = s_abort_raw;
    volatile int *s_odd = s_odd_raw;          // segment (+ 1) that met non-finite values of new rows
    volatile uint8_t *s_skip = s_skip_raw;    // block: halves whose page id is outside the pool
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_launch();
    const int total = tree_total(A, lane, blockIdx.x == 0 && warp == 0);
    const int quota = tree_quota(A, total);
    const int64_t u0l = (int64_t)quota * blockIdx.x;
    if (u0l >= total) return;
    const int u0 = (int)u0l, u1 = min(total - u0, quota) + u0;
    uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *sQ = sm;                                         // high parts, then low parts
    uint8_t *sK = sQ + (C::QLO ? 2 : 1) * C::Q_BYTES;         // [stage]
    uint8_t *sV = sK + ST * C::KV_BYTES;                      // [stage]: dims 0..63, then 64..127
    uint8_t *sP = sV + ST * C::KV_BYTES;                      // [buffer][high, low]
    if (threadIdx.x == 0) {
        for (int i = 0; i < ST; i++) {
            mbar_init(&k_full[i], 1);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_full[i], 1);
            mbar_init(&v_empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&s_full[i], 1);
            mbar_init(&s_free[i], 8);
            mbar_init(&p_full[i], 8);
            mbar_init(&p_free[i], 1);
        }
        mbar_init(&q_full, 8);
        mbar_init(&o_free, 8);
        mbar_init(&fin, 1);
        for (int i = 0; i < 4; i++) mbar_init(&pair_bar[i], 64);
        mbar_fence_init();
        s_abort = 0;
        s_odd[0] = s_odd[1] = 0;
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)),
                     "r"(TR_TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    TreeWalk w;
    w.start(A, u0, u1, lane);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;

    if (warp == 8 || warp == 10) {
        // ---- TMA: K pages (warp 8), V pages (warp 10); the lanes read 32 page ids ahead
        const bool isk = warp == 8;
        uint64_t *full = isk ? k_full : v_full, *empty = isk ? k_empty : v_empty;
        uint8_t *ring = isk ? sK : sV;
        int c = 0;  // blocks issued
        bool ok = true;
        do {
            const int h = w.head(), npg = (w.s.len + PAGE - 1) / PAGE;
            const int32_t *bt = A.bt + (int64_t)w.b * A.max_pages;
            int ids = 0, ids0 = -32;  // this lane's id of page ids0 + lane
            for (int blk = w.blk0; ok && blk < w.blk1; blk++, c++) {
                const int pg0 = blk * PPB;
                if (pg0 >= ids0 + 32 || ids0 < 0) {
                    ids0 = pg0;
                    ids = pg0 + lane < npg ? bt[pg0 + lane] : 0;
                }
                int page[PPB], skip = 0;
#pragma unroll
                for (int i = 0; i < PPB; i++) {
                    page[i] = __shfl_sync(0xffffffffu, ids, pg0 + i - ids0);
                    if (page[i] < 0 || page[i] >= A.num_pages) {  // (pages past the last stand as page 0)
                        skip |= PPB == 1 ? 3 : 1 << i;
                        page[i] = 0;
                    }
                }
                const int st = c % ST;
                if (lane == 0) {
                    if (c >= ST) ok = mbar_wait_bounded(&empty[st], (uint32_t)((c / ST) - 1) & 1u);
                    if (ok) {
                        uint8_t *dst = ring + st * C::KV_BYTES;
                        if (isk) {
                            s_skip[c & 7] = (uint8_t)skip;
                            if (skip) atomicOr(A.err, ERRBIT_BAD_PAGE);
                        }
                        mbar_expect_tx(&full[st], C::KV_BYTES);
#pragma unroll
                        for (int i = 0; i < PPB; i++) {
                            const int row = page[i] * A.n_kv + h;
                            if (isk) {
                                tma_load_2d(dst + i * (HD * PAGE * 2), &kmap, 0, row * HD, &full[st]);
                            } else {
#pragma unroll
                                for (int d = 0; d < HD / 64; d++)
                                    tma_load_2d(dst + d * (TR_KB * 128) + i * (PAGE * 128), &vmap, 64 * d, row * PAGE,
                                                &full[st]);
                            }
                        }
                    }
                }
                ok = __shfl_sync(0xffffffffu, (int)(ok && !s_abort), 0) != 0;
            }
        } while (ok && w.next(A));
        if (lane == 0) {
            if (!ok) s_abort = 1;
            // copies in flight land before shared memory is released
            for (int k = c > ST ? c - ST : 0; k < c; k++) mbar_wait_bounded(&full[k % ST], (uint32_t)(k / ST) & 1u);
        }
    } else if (warp == 9) {
        // ---- MMA issue: S of the next block before O of this one, within a segment
        if (lane == 0) {
            const uint32_t aQ = smem_u32(sQ), aK = smem_u32(sK), aV = smem_u32(sV), aP = smem_u32(sP);
            auto issue_s = [&](int c) -> bool {
                const int st = c % ST, sb = c & 1;
                if (!mbar_wait_bounded(&k_full[st], (uint32_t)(c / ST) & 1u)) return false;
                if (c >= 2 && !mbar_wait_bounded(&s_free[sb], (uint32_t)((c >> 1) - 1) & 1u)) return false;
                tc_fence_after();
#pragma unroll
                for (int ks = 0; ks < HD / 16; ks++) {  // 16 dims: 16 rows of the dim-major pages
                    const uint32_t qo = (uint32_t)(ks >> 2) * (TR_ROWS * 128) + (uint32_t)(ks & 3) * 32;
                    const uint32_t ka = aK + st * C::KV_BYTES + ks * 16 * (PAGE * 2);
                    const uint64_t db = PAGE == 64 ? umma_desc_mn_sw128(ka, C::KV_BYTES, 1024)
                                                   : umma_desc_mn_sw64(ka, HD * PAGE * 2, 512);
                    umma_f16_desc(tmem + sb * TR_KB, umma_desc_sw128(aQ + qo), db, IDESC_S, ks > 0 ? 1u : 0u);
                    if (C::QLO)
                        umma_f16_desc(tmem + sb * TR_KB, umma_desc_sw128(aQ + C::Q_BYTES + qo), db, IDESC_S, 1u);
                }
                umma_commit(&s_full[sb]);
                umma_commit(&k_empty[st]);
                return true;
            };
            auto issue_o = [&](int c, bool first) -> bool {
                const int st = c % ST, pb = c & 1;
                if (!mbar_wait_bounded(&p_full[pb], (uint32_t)(c >> 1) & 1u)) return false;
                if (!mbar_wait_bounded(&v_full[st], (uint32_t)(c / ST) & 1u)) return false;
                tc_fence_after();
                const uint32_t ph = aP + pb * 2 * C::P_BYTES, pl = ph + C::P_BYTES;
#pragma unroll
                for (int ks = 0; ks < TR_KB / 16; ks++) {  // 16 keys
                    const uint64_t db = umma_desc_mn_sw128(aV + st * C::KV_BYTES + ks * 2048, TR_KB * 128, 1024);
                    umma_f16_desc(tmem + TR_O_COL, umma_desc_sw128(ph + ks * 32), db, IDESC_O,
                                  (!first || ks > 0) ? 1u : 0u);
                    umma_f16_desc(tmem + TR_O_COL, umma_desc_sw128(pl + ks * 32), db, IDESC_O, 1u);
                }
                umma_commit(&v_empty[st]);
                umma_commit(&p_free[pb]);
                return true;
            };
            bool ok = true;
            int c = 0, seg = 0;
            do {
                ok = mbar_wait_bounded(&q_full, (uint32_t)seg & 1u) && issue_s(c);
                for (int blk = w.blk0; ok && blk < w.blk1 && !s_abort; blk++, c++) {
                    if (blk + 1 < w.blk1) ok = issue_s(c + 1);
                    if (ok && blk == w.blk0 && seg > 0) ok = mbar_wait_bounded(&o_free, (uint32_t)(seg - 1) & 1u);
                    if (ok) ok = issue_o(c, blk == w.blk0);
                }
                seg++;
            } while (ok && !s_abort && w.next(A));
            if (!ok) s_abort = 1;
            umma_commit(&fin);  // every MMA issued has completed before TMEM is released
            mbar_wait_bounded(&fin, 0);
        }
    } else {
        // ---- softmax: thread = row r (TMEM lane) x 32 key columns
        constexpr unsigned FULL = 0xffffffffu;
        const int qd = warp & 3, ch = warp >> 2, r = 32 * qd + lane;
        const uint32_t lt = tmem + ((uint32_t)(32 * qd) << 16);
        uint32_t npair = 0;  // uses of pair_bar[qd]
        bool ok = true;
        float sl2 = 0.f;     // this row's score unit: scale log2(e) 2^e
        int c = 0, seg = 0;
        auto pair_sync = [&]() -> bool {
            mbar_arrive(&pair_bar[qd]);
            return mbar_wait_bounded(&pair_bar[qd], npair++ & 1u);
        };
        // this thread's half of row r of a group's queries, as fp16 parts scaled by 2^-e
        auto load_q = [&](const TreeWalk &t) -> bool {
            const int rows = t.rows(A);
            if (rows > 32 * qd) {
                const int rr = t.row0() + min(r, rows - 1);
                const T *src = static_cast<const T *>(A.q) + (int64_t)(t.s.off + rr / A.group) * A.qt +
                               (int64_t)(t.head() * A.group + rr % A.group) * HD + ch * (HD / 2);
                float x[HD / 16][8], mx = 0.f;
#pragma unroll
                for (int k = 0; k < HD / 16; k++) tr_load8(src + 8 * k, A.qvec, x[k]);
#pragma unroll
                for (int k = 0; k < HD / 16; k++)
#pragma unroll
                    for (int e = 0; e < 8; e++) mx = fmaxf(mx, fabsf(x[k][e]));
                s_qe[ch][r] = (uint8_t)((__float_as_uint(mx) >> 23) & 255u);
                if (!pair_sync()) return false;
                // exponent that brings the row's largest value to 2^13..2^14 (0 and non-finite rows stay)
                const int ex = max((int)s_qe[0][r], (int)s_qe[1][r]);
                const int e = (ex == 0 || ex == 255) ? 0 : ex - 127 - 13;
                // 2^-e in two factors: e reaches -139 and 114
                const float d0 = __uint_as_float((uint32_t)(127 - e / 2) << 23);
                const float d1 = __uint_as_float((uint32_t)(127 - (e - e / 2)) << 23);
                const float u0f = __uint_as_float((uint32_t)(127 + e / 2) << 23);
                const float u1f = __uint_as_float((uint32_t)(127 + (e - e / 2)) << 23);
                sl2 = __fmul_rn(__fmul_rn(__fmul_rn(A.scale, 1.4426950408889634f), u0f), u1f);
#pragma unroll
                for (int k = 0; k < HD / 16; k++) {
#pragma unroll
                    for (int i = 0; i < 8; i++) x[k][i] = __fmul_rn(__fmul_rn(x[k][i], d0), d1);
                    const int cc = ch * (HD / 16) + k;
                    const uint32_t off = (uint32_t)(cc >> 3) * (TR_ROWS * 128) + sw128_off(r, cc & 7);
                    uint4 hi, lo;
                    split8(x[k], hi, lo);
                    *reinterpret_cast<uint4 *>(sQ + off) = hi;
                    if (C::QLO) *reinterpret_cast<uint4 *>(sQ + C::Q_BYTES + off) = lo;
                }
                fence_proxy_async_smem();  // the tensor core reads them through the async proxy
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full);
            return true;
        };
        ok = load_q(w);
        bool more = ok;
        while (more) {
            const int rows = w.rows(A), pre = w.s.len - w.s.n;
            const bool active = rows > 32 * qd;
            const int rr = w.row0() + min(r, rows - 1), tok = rr / A.group;
            float m = TR_NONE, l = 0.f;
            for (int blk = w.blk0; blk < w.blk1; blk++, c++) {
                const int sb = c & 1, p0 = blk * TR_KB;
                if (!(ok = mbar_wait_bounded(&s_full[sb], (uint32_t)(c >> 1) & 1u))) break;
                tc_fence_after();
                const int skip = s_skip[c & 7];
                float x[32];
                float bm = TR_NONE;
                if (active) {
                    // row maximum of the other half's columns, then this warp's own
                    const bool all = p0 + TR_KB <= pre && !skip;
                    const uint32_t vis = all ? FULL : (skip >> ch) & 1 ? 0u : tree_visible(A, w.s, tok, p0 + 32 * ch);
                    const uint32_t viso =
                        all ? FULL : (skip >> (ch ^ 1)) & 1 ? 0u : tree_visible(A, w.s, tok, p0 + 32 * (ch ^ 1));
                    uint32_t sv[32];
                    tmem_ld32(lt + sb * TR_KB + 32 * (ch ^ 1), sv);
                    if (all) {
#pragma unroll
                        for (int t = 0; t < 32; t++) bm = fmaxf(bm, __fmul_rn(__uint_as_float(sv[t]), sl2));
                    } else {
#pragma unroll
                        for (int t = 0; t < 32; t++)
                            bm = fmaxf(bm, (viso >> t) & 1 ? __fmul_rn(__uint_as_float(sv[t]), sl2) : -INFINITY);
                    }
                    tmem_ld32(lt + sb * TR_KB + 32 * ch, sv);
#pragma unroll
                    for (int t = 0; t < 32; t++) {
                        x[t] = __fmul_rn(__uint_as_float(sv[t]), sl2);
                        if (!all && !((vis >> t) & 1)) x[t] = -INFINITY;
                        bm = fmaxf(bm, x[t]);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&s_free[sb]);  // the MMA of block c + 2 may overwrite it
                if (active) {
                    const float mn = fmaxf(m, bm);
                    const bool need = blk > w.blk0 && mn > m + 8.f;
                    if (__any_sync(FULL, need)) {
                        // rescale this warp's half of the accumulator rows once O of block c - 1 has landed
                        if (!(ok = mbar_wait_bounded(&p_free[sb ^ 1], (uint32_t)((c - 1) >> 1) & 1u))) break;
                        tc_fence_after();
                        const float al = need ? exp2_approx(__fsub_rn(m, mn)) : 1.f;
#pragma unroll 1
                        for (int k = 0; k < HD / 64; k++) {
                            uint32_t ov[32];
                            tmem_ld32(lt + TR_O_COL + (HD / 2) * ch + 32 * k, ov);
#pragma unroll
                            for (int i = 0; i < 32; i++) ov[i] = __float_as_uint(__fmul_rn(__uint_as_float(ov[i]), al));
                            tmem_st32(lt + TR_O_COL + (HD / 2) * ch + 32 * k, ov);
                        }
                        tc_fence_before();
                        if (need) {
                            l = __fmul_rn(l, al);
                            m = mn;
                        }
                    }
                    if (blk == w.blk0) m = mn;
                }
                if (c >= 2 && !(ok = mbar_wait_bounded(&p_free[sb], (uint32_t)((c >> 1) - 1) & 1u))) break;
                if (active) {
                    // p = 2^(x - m + 7), as fp16 high / low A operands
                    const float ref = __fsub_rn(m, TR_LIFT);
                    uint8_t *ph = sP + sb * 2 * C::P_BYTES, *pl = ph + C::P_BYTES;
                    float ls = 0.f;
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        float p[8];
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            p[e] = exp2_approx(__fsub_rn(x[8 * k + e], ref));
                            ls = __fadd_rn(ls, p[e]);
                        }
                        uint4 hi, lo;
                        split8(p, hi, lo);
                        *reinterpret_cast<uint4 *>(ph + sw128_off(r, 4 * ch + k)) = hi;
                        *reinterpret_cast<uint4 *>(pl + sw128_off(r, 4 * ch + k)) = lo;
                    }
                    l = __fadd_rn(l, ls);
                }
                if (p0 + TR_KB > pre || skip) {
                    // Values that some row must not see: 0 * NaN would reach it.  Behind the last key and in
                    // skipped pages all are zeroed; at new rows the non-finite ones, which the rows that see
                    // them get back at the end (s_odd).
                    const int st = c % ST;
                    if (!(ok = mbar_wait_bounded(&v_full[st], (uint32_t)(c / ST) & 1u))) break;
                    for (int i = threadIdx.x; i < (int)C::KV_BYTES / 16; i += 256) {
                        const int t = (i >> 3) & 63;
                        uint4 *cell = reinterpret_cast<uint4 *>(sV + st * C::KV_BYTES) + i;
                        if (p0 + t >= w.s.len || ((skip >> (t >> 5)) & 1)) {
                            *cell = make_uint4(0, 0, 0, 0);
                        } else if (p0 + t >= pre) {
                            uint4 v = *cell;
                            uint32_t *e = reinterpret_cast<uint32_t *>(&v);
                            bool odd = false;
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                if ((e[k] & 0x7C00u) == 0x7C00u) {
                                    e[k] &= 0xffff0000u;
                                    odd = true;
                                }
                                if ((e[k] & 0x7C000000u) == 0x7C000000u) {
                                    e[k] &= 0xffffu;
                                    odd = true;
                                }
                            }
                            if (odd) {
                                *cell = v;
                                s_odd[seg & 1] = seg + 1;
                            }
                        }
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[sb]);
            }
            if (!ok) break;
            // the next group's queries go in while this group's last product runs
            TreeWalk nw = w;
            more = nw.next(A);
            if (more && !(ok = load_q(nw))) break;
            // ---- this segment's rows, once its last product has landed
            if (!(ok = mbar_wait_bounded(&p_free[(c - 1) & 1], (uint32_t)((c - 1) >> 1) & 1u))) break;
            tc_fence_after();
            if (active) {
                s_l[ch][r] = l;
                if (!(ok = pair_sync())) break;
                l = __fadd_rn(s_l[0][r], s_l[1][r]);
                const bool odd = s_odd[seg & 1] == seg + 1;
                const bool whole = !A.split || w.whole();
                const float inv = l > 0.f ? __fdiv_rn(1.f, l) : 0.f;
                float *part = A.part + (int64_t)(2 * blockIdx.x + (seg > 0)) * (HD + 2) * A.rows_cap;
                const int h = w.head();
                T *orow = static_cast<T *>(A.out) + (int64_t)(w.s.off + tok) * A.ot +
                          (int64_t)(h * A.group + rr % A.group) * HD;
#pragma unroll 1
                for (int k = 0; k < HD / 64; k++) {
                    uint32_t ov[32];
                    const int d0 = (HD / 2) * ch + 32 * k;
                    tmem_ld32(lt + TR_O_COL + d0, ov);
                    if (odd) {
                        for (int j = max(0, w.blk0 * TR_KB - pre); j < min(w.s.n, w.blk1 * TR_KB - pre); j++) {
                            const int p = pre + j, page = A.bt[(int64_t)w.b * A.max_pages + p / PAGE];
                            if (page < 0 || page >= A.num_pages || !(tree_visible(A, w.s, tok, p) & 1)) continue;
                            const __half *v = A.vpool + (((int64_t)page * A.n_kv + h) * PAGE + p % PAGE) * HD + d0;
#pragma unroll
                            for (int i = 0; i < 32; i++) {
                                const float x = __half2float(v[i]);
                                if (!isfinite(x)) ov[i] = __float_as_uint(__fadd_rn(__uint_as_float(ov[i]), x));
                            }
                        }
                    }
                    if (!whole) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4)  // [dim / 4][row]: a warp stores 512 bytes at once
                            reinterpret_cast<uint4 *>(part)[(int64_t)((d0 + i) >> 2) * A.rows_cap + r] =
                                make_uint4(ov[i], ov[i + 1], ov[i + 2], ov[i + 3]);
                    } else if (r < rows) {
#pragma unroll
                        for (int i = 0; i < 32; i += 8) {
                            float y[8];
#pragma unroll
                            for (int e = 0; e < 8; e++) y[e] = __fmul_rn(__uint_as_float(ov[i + e]), inv);
                            tr_store8(orow + d0 + i, A.ovec, y);
                        }
                    }
                }
                if (!whole && ch == 0)
                    reinterpret_cast<float2 *>(part + (int64_t)HD * A.rows_cap)[r] = make_float2(m, l);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&o_free);
            w = nw;
            seg++;
        }
        if (!ok) s_abort = 1;
    }
    tc_fence_before();
    __syncthreads();
    if (s_abort && threadIdx.x == 0) atomicOr(A.err, ERRBIT_WAIT_TIMEOUT);
    if (warp == 9) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TR_TMEM_COLS)
                     : "memory");
    }
}

// Joins the partials of the groups that several CTAs hold.  grid (row tiles a
// sequence x rows_cap / 32 x dim quarters, n_kv, batch): lane = row, warp =
// HD / 64 four-dim columns.
template <typename T, int HD>
__global__ void __launch_bounds__(128) k_attn_tree_join(const __grid_constant__ TreeArgs A) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int quarter = blockIdx.x & 3, rest = blockIdx.x >> 2;
    const int slabs = A.rows_cap / 32, slab = rest % slabs, tile = rest / slabs;
    const int b = blockIdx.z;
    TreeSeq s;
    s.load(A, b);
    const int row0 = tile * TR_ROWS + 32 * slab;
    if (row0 >= s.n * A.group) return;
    // units before this sequence, and in all
    int before = 0, total = 0;
    for (int i = lane; i < A.batch; i += 32) {
        TreeSeq o;
        o.load(A, i);
        const int u = o.units(A);
        total += u;
        if (i < b) before += u;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        total += __shfl_xor_sync(0xffffffffu, total, o);
        before += __shfl_xor_sync(0xffffffffu, before, o);
    }
    const int quota = tree_quota(A, total);
    const int gs = before + (blockIdx.y * s.tiles + tile) * s.blocks, ge = gs + s.blocks;  // the group's units
    const int c0 = gs / quota, c1 = (ge - 1) / quota;
    if (c0 == c1) return;  // written by its CTA
    const int r = 32 * slab + lane;
    const int64_t slot = (int64_t)(HD + 2) * A.rows_cap;
    // a CTA's first segment is its partial 0: every one but the first CTA's starts with this group
    auto part = [&](int c) { return A.part + (2 * (int64_t)c + (c * (int64_t)quota < gs)) * slot; };
    pdl_wait();
    float M = TR_NONE;
    for (int c = c0; c <= c1; c++) M = fmaxf(M, reinterpret_cast<const float2 *>(part(c) + (int64_t)HD * A.rows_cap)[r].x);
    float L = 0.f;
    constexpr int N = HD / 64;  // float4 columns a thread
    float4 o[N];
#pragma unroll
    for (int k = 0; k < N; k++) o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    const int col0 = quarter * (HD / 16) + warp * N;
#pragma unroll 4
    for (int c = c0; c <= c1; c++) {
        const float *p = part(c);
        const float2 ml = reinterpret_cast<const float2 *>(p + (int64_t)HD * A.rows_cap)[r];
        const float wgt = exp2f(__fsub_rn(ml.x, M));
        L = __fmaf_rn(wgt, ml.y, L);
#pragma unroll
        for (int k = 0; k < N; k++) {
            const float4 v = reinterpret_cast<const float4 *>(p)[(int64_t)(col0 + k) * A.rows_cap + r];
            o[k].x = __fmaf_rn(wgt, v.x, o[k].x);
            o[k].y = __fmaf_rn(wgt, v.y, o[k].y);
            o[k].z = __fmaf_rn(wgt, v.z, o[k].z);
            o[k].w = __fmaf_rn(wgt, v.w, o[k].w);
        }
    }
    const int rr = row0 + lane;
    if (rr >= s.n * A.group) return;
    const float inv = L > 0.f ? __fdiv_rn(1.f, L) : 0.f;
    T *out = static_cast<T *>(A.out) + (int64_t)(s.off + rr / A.group) * A.ot +
             (int64_t)(blockIdx.y * A.group + rr % A.group) * HD + 4 * col0;
#pragma unroll
    for (int k = 0; k < N; k++) {
        tr_put(out + 4 * k, __fmul_rn(o[k].x, inv));
        tr_put(out + 4 * k + 1, __fmul_rn(o[k].y, inv));
        tr_put(out + 4 * k + 2, __fmul_rn(o[k].z, inv));
        tr_put(out + 4 * k + 3, __fmul_rn(o[k].w, inv));
    }
}

// What a call of these sizes launches.
struct TreePlan {
    int split, ctas, rows_cap, tiles;
    int64_t ws;
};
static TreePlan tree_plan(const fb_ctx *ctx, int batch, int max_new, int n_heads, int n_kv, int head_dim,
                          int max_seq_len) {
    TreePlan p{};
    const int64_t rows = (int64_t)max_new * (n_heads / n_kv);
    const int64_t tiles = (rows + TR_ROWS - 1) / TR_ROWS, blocks = (max_seq_len + TR_KB - 1) / TR_KB;
    const int64_t groups = tiles * n_kv * batch;
    FB_REQUIRE(groups * blocks < ((int64_t)1 << 31) - 4096 && tiles <= 65535, "attn_tree: batch too large");
    p.split = blocks > TR_WHOLE;
    const int64_t units = p.split ? groups * blocks : groups;
    p.ctas = (int)(units < ctx->num_sms ? units : ctx->num_sms);
    p.tiles = (int)tiles;
    p.rows_cap = (int)(rows >= TR_ROWS ? TR_ROWS : (rows + 31) / 32 * 32);
    p.ws = p.split ? (int64_t)2 * p.ctas * (head_dim + 2) * p.rows_cap * 4 : 0;
    return p;
}

template <typename T, int HD, int PAGE>
static void launch_tree(fb_ctx *ctx, const TreeArgs &A, const TreePlan &plan, const CUtensorMap &kmap,
                        const CUtensorMap &vmap) {
    constexpr size_t smem = TreeCfg<T, HD>::SMEM;
    FB_CUDA(cudaFuncSetAttribute(k_attn_tree<T, HD, PAGE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    k_attn_tree<T, HD, PAGE><<<plan.ctas, TR_THREADS, smem, ctx->stream>>>(kmap, vmap, A);
    FB_CUDA(cudaGetLastError());
    if (!plan.split) return;
    // the join's blocks start while the attention drains and wait for it (programmatic dependent launch)
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = ctx->pdl ? 1 : 0;
    cfg.gridDim = dim3((unsigned)(plan.tiles * (plan.rows_cap / 32) * 4), (unsigned)A.n_kv, (unsigned)A.batch);
    cfg.blockDim = dim3(128);
    cfg.stream = ctx->stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    FB_CUDA(cudaLaunchKernelEx(&cfg, k_attn_tree_join<T, HD>, A));
}

static void check_tree_shape(int batch, int max_new, int n_heads, int n_kv, int head_dim, int page_size,
                             int max_seq_len) {
    FB_REQUIRE(head_dim == 64 || head_dim == 128, "attn_tree: head_dim must be 64 or 128");
    FB_REQUIRE(page_size == 32 || page_size == 64, "attn_tree: page_size must be 32 or 64");
    FB_REQUIRE(batch >= 0 && batch <= 65535 && max_new >= 0 && n_heads >= 1 && n_kv >= 1 && n_heads <= 65535 &&
                   max_seq_len >= 0 && max_seq_len <= 1 << 30,
               "attn_tree: bad shape");
    FB_REQUIRE(n_heads % n_kv == 0, "attn_tree: n_heads must be a multiple of n_kv_heads");
}

}  // namespace fb

using namespace fb;

extern "C" {

int fb_attn_tree_workspace(fb_ctx *ctx, int batch, int max_new, int n_heads, int n_kv_heads, int head_dim,
                           int page_size, int max_seq_len, int64_t *bytes) {
    return guarded([&] {
        check_tree_shape(batch, max_new, n_heads, n_kv_heads, head_dim, page_size, max_seq_len);
        FB_REQUIRE(ctx && bytes, "null argument");
        *bytes = batch && max_new && max_seq_len
                     ? tree_plan(ctx, batch, max_new, n_heads, n_kv_heads, head_dim, max_seq_len).ws
                     : 0;
    });
}

int fb_attn_tree(fb_ctx *ctx, int dtype, const void *q_dev, int64_t q_token_stride, const void *k_pages_dev,
                 const void *v_pages_dev, const int32_t *block_table_dev, const int32_t *row_offsets_dev,
                 const int32_t *seq_lens_dev, const uint32_t *mask_dev, int mask_words, void *out_dev,
                 int64_t out_token_stride, int batch, int n_rows, int max_new, int n_heads, int n_kv_heads,
                 int head_dim, int page_size, int max_pages, int num_pages, int max_seq_len, float scale,
                 void *workspace_dev, int64_t workspace_bytes) {
    return guarded([&] {
        FB_REQUIRE(dtype == FB_F32 || dtype == FB_F16 || dtype == FB_BF16,
                   "attn_tree: dtype must be FB_F32, FB_F16 or FB_BF16");
        check_tree_shape(batch, max_new, n_heads, n_kv_heads, head_dim, page_size, max_seq_len);
        FB_REQUIRE(n_rows >= 0 && max_pages >= 1 && num_pages >= 1, "attn_tree: bad shape");
        FB_REQUIRE(max_seq_len <= (int64_t)max_pages * page_size, "attn_tree: max_seq_len exceeds the block table");
        FB_REQUIRE(!mask_dev || mask_words >= (max_new + 31) / 32, "attn_tree: mask_words is below max_new / 32");
        FB_REQUIRE(q_token_stride >= 0 && (n_rows <= 1 || out_token_stride >= (int64_t)n_heads * head_dim),
                   "attn_tree: bad token stride");
        FB_REQUIRE(isfinite(scale), "attn_tree: scale must be finite");
        if (batch == 0 || n_rows == 0 || max_new == 0 || max_seq_len == 0) return;
        FB_REQUIRE(ctx && q_dev && k_pages_dev && v_pages_dev && block_table_dev && row_offsets_dev && seq_lens_dev &&
                       out_dev,
                   "null argument");
        const size_t esz = dtype == FB_F32 ? 4 : 2;
        FB_REQUIRE((((uintptr_t)q_dev | (uintptr_t)out_dev) & (esz - 1)) == 0 &&
                       (((uintptr_t)row_offsets_dev | (uintptr_t)seq_lens_dev | (uintptr_t)block_table_dev |
                         (uintptr_t)mask_dev) & 3) == 0,
                   "attn_tree: misaligned pointer");
        FB_REQUIRE((((uintptr_t)k_pages_dev | (uintptr_t)v_pages_dev) & 15) == 0,
                   "attn_tree: KV pools must be 16-byte aligned");
        DeviceGuard guard(ctx->device);
        TreeArgs A{};
        A.q = q_dev;
        A.qt = q_token_stride;
        A.ot = out_token_stride;
        A.kpool = static_cast<const __half *>(k_pages_dev);
        A.vpool = static_cast<const __half *>(v_pages_dev);
        A.bt = block_table_dev;
        A.offsets = row_offsets_dev;
        A.lens = seq_lens_dev;
        A.mask = mask_dev;
        A.mask_words = mask_words;
        A.out = out_dev;
        A.batch = batch;
        A.n_rows = n_rows;
        A.max_new = max_new;
        A.n_heads = n_heads;
        A.n_kv = n_kv_heads;
        A.max_pages = max_pages;
        A.num_pages = num_pages;
        A.max_seq = max_seq_len;
        A.scale = scale;
        A.err = ctx->err_word;
        const TreePlan plan = tree_plan(ctx, batch, max_new, n_heads, n_kv_heads, head_dim, max_seq_len);
        FB_REQUIRE(plan.ws == 0 || (workspace_dev && workspace_bytes >= plan.ws && ((uintptr_t)workspace_dev & 15) == 0),
                   "attn_tree: the workspace must be 16-byte aligned and hold fb_attn_tree_workspace bytes (" +
                       std::to_string(plan.ws) + ")");
        A.group = n_heads / n_kv_heads;
        A.split = plan.split;
        A.ctas = plan.ctas;
        A.rows_cap = plan.rows_cap;
        A.part = static_cast<float *>(workspace_dev);
        const int V = (int)(16 / esz);
        A.qvec = ((uintptr_t)q_dev & 15) == 0 && q_token_stride % V == 0;
        A.ovec = ((uintptr_t)out_dev & 15) == 0 && out_token_stride % V == 0;
        FB_REQUIRE((int64_t)num_pages * n_kv_heads * head_dim < ((int64_t)1 << 31), "attn_tree: KV pool too large");
        const CUtensorMap kmap = pool_map("attn_tree", k_pages_dev, (int64_t)num_pages * n_kv_heads * head_dim,
                                          page_size, (uint32_t)page_size, (uint32_t)head_dim);
        const CUtensorMap vmap = pool_map("attn_tree", v_pages_dev, (int64_t)num_pages * n_kv_heads * page_size,
                                          head_dim, 64, (uint32_t)page_size);
        auto go = [&](auto t) {
            using T = decltype(t);
            if (head_dim == 128 && page_size == 64) launch_tree<T, 128, 64>(ctx, A, plan, kmap, vmap);
            else if (head_dim == 128) launch_tree<T, 128, 32>(ctx, A, plan, kmap, vmap);
            else if (page_size == 64) launch_tree<T, 64, 64>(ctx, A, plan, kmap, vmap);
            else launch_tree<T, 64, 32>(ctx, A, plan, kmap, vmap);
        };
        if (dtype == FB_F32) go(float{});
        else if (dtype == FB_F16) go(__half{});
        else go(__nv_bfloat16{});
    });
}

}  // extern "C"
