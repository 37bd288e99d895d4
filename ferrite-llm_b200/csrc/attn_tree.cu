// Attention of drafted token trees over the paged cache (fb_attn_tree).  No
// reference counterpart: the reference verifies one chain, token by token
// (crates/ferrite-core/src/generation.rs:340-535).
//
// o = sum_j p_j v_j / sum_j p_j, p_j = exp(scale q.k_j - m), j over the prefix
// and the drafted tokens whose mask bit is set.
//
// The (drafted token, query head of the group) pairs of a sequence and kv head
// are the rows of one matrix product, up to 256 rows a group (two tiles of 128,
// the MMA's M; f32: one): they share every key and value that is read.  A verified tree of
// 32 tokens with 4 heads a kv head needs 128 multiplications a byte of cache, so
// up to one full tile the bound is HBM (4 head_dim bytes a key and kv head),
// beyond it the tensor cores.
//
// Split: the (sequence, kv head, row group, 64-key block) units of a call (two
// for a block that two tiles work on) are counted on the device from the lengths
// and dealt to one CTA per SM in equal contiguous shares, so unequal lengths and
// few sequences fill the machine alike.  A row group that one CTA holds whole is
// written directly; the others leave (max, sum, o) partials, at most two a CTA,
// that a second kernel joins in share order (no atomics: the same bits every
// time).  Calls of at most TR_WHOLE blocks a group deal whole groups, unjoined.
//
// A CTA, 12 warps: two softmax groups of 4 warps (thread = row), 8 and 10 TMA
// copies of K and V pages, 9 and 11 issue tcgen05.mma for a group each (9 owns the
// tensor memory).  For 16-bit
// results: with more than 128 rows each softmax group has a tile and both read
// the same keys; otherwise they take the blocks of one tile in turn, each with its
// own running maximum, sum and accumulator, merged at the end.  Either way one
// group's products run under the other's exponentials, which no single chain of
// blocks could hide.  For f32 results: one tile, one group takes the exponentials
// and the other the products (below).  The dim-major K pages and token-major V pages land in shared
// memory as the MN-major operands of S = Q K^T and O += P V; the probabilities
// replace the scores in tensor memory and are the A operand from there.  Scores
// have two buffers a group.  The roles run on through the CTA's groups: the next
// group's keys load while one drains.
//
// Precision: q is scaled by a power of two a row (to 2^13..2^14 at most) and
// enters as fp16 high + low parts where it is f32 (f16 and bf16 queries fit the
// high part); the probabilities are kept 2^7 above the running maximum's unit (at
// most 2^15).  For f32 and f16 results they are fp16 high + low parts, 22 bits down
// to 2^-21 of the largest: f16 results are off by their own rounding alone (1.37
// times that with the high part alone; the second product costs 2.5 us of 45 below).
// For bf16 results the high part is enough: it is off by 2^-11 of a probability
// where a result's own rounding is 2^-8 of it (together 1.008 times that rounding
// in the 2-norm; the low part would cost a fifth of the long contexts' time below).
// Products and sums are f32.  The tensor core truncates its sums, by 2^-25 of
// them on average at each instruction, always towards zero: over 100 blocks that
// is 10^-5 (7.4e-6 measured in the 2-norm at 30000 keys), little beside a 16-bit
// result's rounding, but not beside f32's.  So f32 results have each block's product
// start from zero and the second group adds it to its registers, a rounded FMA an
// element (6.6e-7 there).  Where the tensor core does accumulate, the sums are
// rescaled only when a row's maximum grows by more than 8 (log 2 units).
//
// Measured (back to back in a graph, the join included; 6559 GB/s the copy rate,
// 1627 TFLOP/s the library's bf16 rate): 16 sequences of 25 new rows over up to
// 4096 keys, 32 heads on 8, f16: 45.2 us, 4.0 TB/s of keys and values; 4 of 40
// over 32000, 64 heads, bf16: 154 us, 640 TFLOP/s, where the exponentials and the
// 64-key products (N = 64 runs at two thirds of N = 128's rate) take turns; 60 rows
// over 4096, f32: 27.4 us, half of it the queries' way in and the join; 7 over 190:
// 12.4 us, three blocks and the same ends.
#include <math.h>

#include <type_traits>

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
    uint64_t inv_group;  // ceil(2^32 / group)
    int split;      // 1: units are key blocks, 0: whole groups
    int ctas;       // CTAs of the attention kernel
    int grows;      // rows a group: 128 (f32) or 256
    int rows_cap;   // row capacity of a partial (multiple of 32, <= 256)
    float *part;    // [2 ctas] partials of (head_dim + 2) rows_cap floats
    float scale;
    bool qvec, ovec;  // q / out rows start on 16 bytes
    uint32_t *err;
};

constexpr int TR_ROWS = 128;      // rows a tile (MMA M)
constexpr int TR_PAIR = 256;      // rows a group at most: two tiles
constexpr int TR_KB = 64;         // keys a block
constexpr int TR_WHOLE = 4;
constexpr int TR_SWITCH = 8;
constexpr int TR_THREADS = 384;
constexpr float TR_NONE = -3e38f;  // running maximum of a row that has seen nothing
constexpr float TR_LIFT = 7.f;     // probabilities are kept 2^7 above the reference maximum
constexpr float TR_FAR = 1048576.f;  // 2^20: maxima beyond it are taken off the scores before the lift is added

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

// One sequence of the batch: its new rows, key blocks, row groups a kv head (the
// last of `weight` units a block, the others of `full`).  A sequence left out has
// none.
struct TreeSeq {
    int off, n, len, blocks, pairs, weight, full;
    __device__ __forceinline__ bool load(const TreeArgs &A, int b) {
        off = A.offsets[b];
        n = A.offsets[b + 1] - off;
        len = A.lens[b];
        const bool ok = off >= 0 && n >= 0 && n <= A.max_new && off <= A.n_rows - n && len >= n && len <= A.max_seq;
        if (!ok) n = len = 0;
        blocks = (len + TR_KB - 1) / TR_KB;
        const int rows = n * A.group;
        full = A.grows / TR_ROWS;
        pairs = (rows + A.grows - 1) / A.grows;
        weight = rows - (pairs - 1) * A.grows > TR_ROWS ? 2 : 1;
        return ok;
    }
    __device__ __forceinline__ int per(const TreeArgs &A) const { return A.split ? blocks : 1; }
    __device__ __forceinline__ int head_units(const TreeArgs &A, int lead) const {
        return pairs > 0 ? (full * (pairs - 1) + weight) * per(A) + pairs * lead : 0;
    }
    __device__ __forceinline__ int units(const TreeArgs &A, int lead) const { return head_units(A, lead) * A.n_kv; }
    __device__ __forceinline__ int groups(const TreeArgs &A) const { return pairs * A.n_kv; }
};

// Units of all sequences without leads, and row groups: the warp's sums.
struct TreeTotal {
    int units, groups;
    __device__ __forceinline__ void add(const TreeArgs &A, const TreeSeq &s) {
        units += s.units(A, 0);
        groups += s.groups(A);
    }
    __device__ __forceinline__ void reduce() {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            units += __shfl_xor_sync(0xffffffffu, units, o);
            groups += __shfl_xor_sync(0xffffffffu, groups, o);
        }
    }
    // Units that a row group has in front of its blocks: what it costs a CTA to begin another one (its queries wait for
    // the last scores, its rows are written out), so that the shares with a border inside hold fewer blocks.  Where no
    // CTA has more than a unit there is no border.  (When it was chosen: 60 new rows of 32 heads at 4096 keys, f32: 26.6
    // us; 29.1 with 3, 32.7 with none; 16 sequences of 25 rows, f16: 43.2, 44.4, 47.3.)
    __device__ __forceinline__ int lead(const TreeArgs &A) const { return A.split && units > A.ctas ? TR_SWITCH : 0; }
    // A CTA's share; the join kernel derives the same one.  With split and blocks of two units at least two, so that
    // none lies inside such a block.
    __device__ __forceinline__ int all(const TreeArgs &A) const { return units + groups * lead(A); }
    __device__ __forceinline__ int quota(const TreeArgs &A) const {
        return max(A.split && A.grows > TR_ROWS ? 2 : 1, (all(A) + A.ctas - 1) / A.ctas);
    }
};

// The segments of a CTA's share: consecutive blocks of one row group.  A block
// (without split: a group) belongs to the share that holds its first unit.
struct TreeWalk {
    TreeSeq s;
    int b, h, pair, blk0, blk1, left, lead;
    // warp-collective; this CTA's share.  False: it holds no block's first unit.
    __device__ __forceinline__ bool start(const TreeArgs &A, int cta, int lane, bool report) {
        int base = 0, mine = 0;
        TreeTotal t{};
        s = TreeSeq{};
        for (int i = lane; i < A.batch; i += 32) {
            TreeSeq o;
            if (!o.load(A, i) && report) atomicOr(A.err, ERRBIT_BAD_POS);
            t.add(A, o);
            if (i < 32) s = o;  // (the first 32 sequences stay in the lanes' registers)
        }
        const TreeSeq first = s;
        t.reduce();
        lead = t.lead(A);
        const int total = t.all(A), quota = t.quota(A);
        mine = s.units(A, lead);
        const int64_t u0l = (int64_t)quota * cta;
        if (u0l >= total) return false;
        const int u0 = (int)u0l;
        left = min(total - u0, quota);
        b = 0;
        for (int b0 = 0; b0 < A.batch; b0 += 32) {
            if (b0 > 0) {
                mine = 0;
                if (b0 + lane < A.batch) {
                    s.load(A, b0 + lane);
                    mine = s.units(A, lead);
                }
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
        if (b < 32) {
            s.off = __shfl_sync(0xffffffffu, first.off, b);
            s.n = __shfl_sync(0xffffffffu, first.n, b);
            s.len = __shfl_sync(0xffffffffu, first.len, b);
            s.blocks = __shfl_sync(0xffffffffu, first.blocks, b);
            s.pairs = __shfl_sync(0xffffffffu, first.pairs, b);
            s.weight = __shfl_sync(0xffffffffu, first.weight, b);
            s.full = A.grows / TR_ROWS;
        } else {
            s.load(A, b);
        }
        const int each = s.full * s.per(A) + lead, hu = s.head_units(A, lead);
        int r = u0 - base;
        h = r / hu;
        r -= h * hu;
        pair = min(r / each, s.pairs - 1);
        r -= pair * each;
        span(A, r);
        return blk0 < blk1 || next(A);
    }
    __device__ __forceinline__ int weight() const { return pair < s.pairs - 1 ? s.full : s.weight; }
    __device__ __forceinline__ void span(const TreeArgs &A, int r) {
        const int w = weight(), take = min(left, w * s.per(A) + lead - r);
        if (A.split) {
            blk0 = (max(r - lead, 0) + w - 1) / w;
            blk1 = (max(r + take - lead, 0) + w - 1) / w;
        } else {
            blk0 = r == 0 ? 0 : s.blocks;
            blk1 = s.blocks;
        }
        left -= take;
    }
    __device__ __forceinline__ bool next(const TreeArgs &A) {
        do {
            if (left <= 0) return false;
            if (++pair == s.pairs) {
                pair = 0;
                if (++h == A.n_kv) {
                    h = 0;
                    do {
                        if (++b >= A.batch) return false;
                        s.load(A, b);
                    } while (s.groups(A) == 0);
                }
            }
            span(A, 0);
        } while (blk0 >= blk1);
        return true;
    }
    __device__ __forceinline__ int row0(const TreeArgs &A) const { return pair * A.grows; }
    __device__ __forceinline__ int rows(const TreeArgs &A) const { return min(A.grows, s.n * A.group - row0(A)); }
    __device__ __forceinline__ bool both() const { return weight() == 2; }  // two tiles
    // blocks that softmax group g works on
    __device__ __forceinline__ int jobs(int g) const { return both() ? blk1 - blk0 : (blk1 - blk0 + 1 - g) / 2; }
    __device__ __forceinline__ bool whole() const { return blk0 == 0 && blk1 == s.blocks; }
};

// The power of two that a row's queries are divided by, from the exponent field of
// their largest magnitude: it comes to 2^13..2^14 (rows below 2^-107 less, which
// costs them no bit; 0 and non-finite ones stay).
__device__ __forceinline__ int tree_shift(int ex) { return ex == 0 || ex == 255 ? 0 : max(ex - 127 - 13, -120); }

// A row's new row of its sequence: row / group (exact while row group < 2^32).
__device__ __forceinline__ int tree_token(const TreeArgs &A, int row) {
    return (int)(((uint64_t)(uint32_t)row * A.inv_group) >> 32);
}

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
    static constexpr bool LO = sizeof(T) == 4;          // f32: q has low parts, the blocks are summed in registers
    static constexpr bool PLO = !std::is_same<T, __nv_bfloat16>::value;  // the probabilities have low parts
    static constexpr int ST = HD == 128 && LO ? 4 : 5;  // K and V stages
    static constexpr uint32_t Q_BYTES = TR_ROWS * HD * 2;
    static constexpr uint32_t TILE_BYTES = (LO ? 2 : 1) * Q_BYTES;  // a tile's queries
    static constexpr uint32_t KV_BYTES = TR_KB * HD * 2;            // one block of K or V
    static constexpr int TILES = LO ? 1 : 2;  // row tiles a group
    static constexpr size_t SMEM = 1024 + TILES * (size_t)TILE_BYTES + 2 * ST * (size_t)KV_BYTES;
    static_assert(SMEM + (LO ? 5120 : 2048) <= 227 * 1024, "tree attention stages must fit");
};
// Tensor memory columns: scores (group, buffer) at 128 g + 64 buffer, O of group (f32: buffer) g at 256 + HD g.
constexpr uint32_t TR_TMEM_COLS = 512;  
constexpr uint32_t TR_O_COL = 256;

// Bounded wait (~1 s) for waits that are short in the steady state: polls without the suspension of
// mbar_wait_bounded, which a satisfied wait pays for too.
__device__ __forceinline__ bool tr_wait(uint64_t *bar, uint32_t parity) {
    auto poll = [&]() {
        uint32_t ok;
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity)
            : "memory");
        return ok != 0;
    };
    for (int i = 0; i < 16; i++)
        if (poll()) return true;
    return mbar_wait_bounded(bar, parity);
}

// D += A B with A (fp16 pairs, K-major, a lane a row) in tensor memory.
__device__ __forceinline__ void umma_f16_tmem(uint32_t tmem_d, uint32_t tmem_a, uint64_t db, uint32_t idesc,
                                              uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(tmem_d),
        "r"(tmem_a), "l"(db), "r"(idesc), "r"(accumulate)
        : "memory");
}

template <typename T, int HD, int PAGE>
__global__ void __launch_bounds__(TR_THREADS, 1)
    k_attn_tree(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                const __grid_constant__ TreeArgs A) {
    using C = TreeCfg<T, HD>;
    constexpr int ST = C::ST, PPB = TR_KB / PAGE;  // pages a block
    constexpr uint32_t IDESC_S = umma_idesc_f16(TR_ROWS, TR_KB, false, true);
    constexpr uint32_t IDESC_O = umma_idesc_f16(TR_ROWS, HD, false, true);
    extern __shared__ uint8_t smem_raw[];
    // A stage's full barrier alternates between two: a waiter meets its block's phase there without having waited for
    // the block before it in that stage (with one tile the groups take every other block).  The barrier's own last
    // block, 2 ST back, has been consumed by then: a block is loaded only once the one ST back has been.
    __shared__ uint64_t k_full[2 * ST], k_empty[ST], v_full[2 * ST], v_empty[ST];
    __shared__ uint64_t s_full[2][2], p_full[2][2], o_done[2][2];  // [group][buffer]
    __shared__ uint64_t q_full, q_empty, o_free, fin[2], go, pair_bar[4];
    // f32: a block's product has been read; a segment's (max, sum) are there, have been read ([parity])
    __shared__ uint64_t o_read[C::LO ? 2 : 1], ml_full[C::LO ? 2 : 1], ml_read[C::LO ? 2 : 1];
    __shared__ uint32_t s_tmem;
    __shared__ float2 s_ml[C::LO ? 2 : 1][TR_ROWS];  // (max, sum) of a tile's rows: of group 1; f32: [segment parity]
    __shared__ float s_al[C::LO ? 4 : 1][TR_ROWS];   // f32: [job mod 4] what the rows' sums so far are scaled by
    __shared__ uint8_t s_qe[2][TR_PAIR];  // [segment parity] exponent field of a row's largest query value
    __shared__ int s_abort_raw, s_odd_raw[2];
    __shared__ uint8_t s_skip_raw[16];
    volatile int &s_abort = s_abort_raw;
    volatile int *s_odd = s_odd_raw;        // segment (+ 1) that met non-finite values of new rows
    volatile uint8_t *s_skip = s_skip_raw;  // block: halves whose page id is outside the pool
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *sQ = sm;                             // [tile][high parts, low parts]
    uint8_t *sK = sQ + C::TILES * C::TILE_BYTES;  // [stage]
    uint8_t *sV = sK + ST * C::KV_BYTES;          // [stage]: dims 0..63, then 64..127
    if (threadIdx.x == 0) {
        for (int i = 0; i < ST; i++) {
            mbar_init(&k_full[i], 1);
            mbar_init(&k_full[ST + i], 1);
            mbar_init(&k_empty[i], C::LO ? 1 : 2);  // (both MMA warps)
            mbar_init(&v_full[i], 1);
            mbar_init(&v_full[ST + i], 1);
            mbar_init(&v_empty[i], C::LO ? 1 : 2);
        }
        for (int i = 0; i < 4; i++) {
            mbar_init(&s_full[i >> 1][i & 1], 1);
            mbar_init(&p_full[i >> 1][i & 1], 4);
            mbar_init(&o_done[i >> 1][i & 1], 1);
            mbar_init(&pair_bar[i], 32);
        }
        mbar_init(&q_full, 8);
        mbar_init(&go, 8);
        mbar_init(&q_empty, C::LO ? 1 : 2);
        for (int i = 0; i < (C::LO ? 2 : 1); i++) {
            mbar_init(&o_read[i], 4);
            mbar_init(&ml_full[i], 4);
            mbar_init(&ml_read[i], 4);
        }
        mbar_init(&o_free, 8);
        mbar_init(&fin[0], 1);
        mbar_init(&fin[1], 1);
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
    pdl_wait();    // (the set-up above overlaps the predecessor's end)
    pdl_launch();  // (now: the join reads the lengths before it waits)
    TreeWalk w;
    const bool share = w.start(A, blockIdx.x, lane, blockIdx.x == 0 && warp == 0);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;

    if (!share) {
        // nothing to do: straight to the release of the tensor memory
    } else if (warp == 8 || warp == 10) {
        // ---- TMA: K pages (warp 8), V pages (warp 10); the lanes read 32 page ids ahead
        const bool isk = warp == 8;
        uint64_t *full = isk ? k_full : v_full, *empty = isk ? k_empty : v_empty;
        uint8_t *ring = isk ? sK : sV;
        int c = 0;  // blocks issued
        bool ok = true;
        do {
            const int npg = (w.s.len + PAGE - 1) / PAGE;
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
                const int st = c % ST, fb = c % (2 * ST);
                if (lane == 0) {
                    // (the first queries, two dependent steps from the first scores, are not queued behind the rings)
                    if (c == 1) ok = tr_wait(&go, 0);
                    if (c >= ST) ok = ok && tr_wait(&empty[st], (uint32_t)((c / ST) - 1) & 1u);
                    if (ok) {
                        uint8_t *dst = ring + st * C::KV_BYTES;
                        if (isk) {
                            s_skip[c & 15] = (uint8_t)skip;
                            if (skip) atomicOr(A.err, ERRBIT_BAD_PAGE);
                        }
                        mbar_expect_tx(&full[fb], C::KV_BYTES);
#pragma unroll
                        for (int i = 0; i < PPB; i++) {
                            const int row = page[i] * A.n_kv + w.h;
                            if (isk) {
                                tma_load_2d(dst + i * (HD * PAGE * 2), &kmap, 0, row * HD, &full[fb]);
                            } else {
#pragma unroll
                                for (int d = 0; d < HD / 64; d++)
                                    tma_load_2d(dst + d * (TR_KB * 128) + i * (PAGE * 128), &vmap, 64 * d, row * PAGE,
                                                &full[fb]);
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
            for (int k = c > ST ? c - ST : 0; k < c; k++)
                mbar_wait_bounded(&full[k % (2 * ST)], (uint32_t)(k / (2 * ST)) & 1u);
        }
    } else if (C::LO && warp >= 8) {
        // ---- f32, MMA issue (warp 9): the next block's scores before this one's product, which starts from zero in
        // one of two buffers: the tensor core truncates every addition to an accumulator (2^-24 of it), which over a
        // long context would add up, so the blocks are summed with rounding elsewhere.
        if (warp == 9 && lane == 0) {
            const uint64_t dQ = umma_desc_sw128(smem_u32(sQ)), dV = umma_desc_mn_sw128(smem_u32(sV), TR_KB * 128, 1024);
            const uint64_t dK = PAGE == 64 ? umma_desc_mn_sw128(smem_u32(sK), C::KV_BYTES, 1024)
                                           : umma_desc_mn_sw64(smem_u32(sK), HD * PAGE * 2, 512);
            int j = 0, seg = 0;  // blocks of the segments before this one
            bool ok = true;
            auto issue_s = [&](int c) -> bool {
                const int st = c % ST, f = c % (2 * ST);
                const uint32_t d = tmem + TR_KB * (c & 1);
                const uint64_t kd = dK + st * (C::KV_BYTES >> 4);
                if (!tr_wait(&k_full[f], (uint32_t)(c / (2 * ST)) & 1u)) return false;
                tc_fence_after();
#pragma unroll
                for (int i = 0; i < 2 * (HD / 16); i++) {  // the low parts first: small sums lose less
                    const int ks = i % (HD / 16);
                    const uint32_t qo = ((uint32_t)(ks >> 2) * (TR_ROWS * 128) + (uint32_t)(ks & 3) * 32 +
                                         (i < HD / 16 ? C::Q_BYTES : 0)) >> 4;
                    umma_f16_desc(d, dQ + qo, kd + ks * (16 * PAGE * 2 >> 4), IDESC_S, i > 0 ? 1u : 0u);
                }
                umma_commit(&s_full[0][c & 1]);
                umma_commit(&k_empty[st]);
                return true;
            };
            auto issue_o = [&](int c) -> bool {
                const int st = c % ST, f = c % (2 * ST);
                const uint32_t p = tmem + TR_KB * (c & 1), d = tmem + TR_O_COL + HD * (c & 1);
                const uint64_t vd = dV + st * (C::KV_BYTES >> 4);
                if (!tr_wait(&v_full[f], (uint32_t)(c / (2 * ST)) & 1u)) return false;
                if (c >= 2 && !tr_wait(&o_read[c & 1], (uint32_t)((c >> 1) - 1) & 1u)) return false;
                if (!tr_wait(&p_full[0][c & 1], (uint32_t)(c >> 1) & 1u)) return false;
                tc_fence_after();
#pragma unroll
                for (int i = 0; i < 2 * (TR_KB / 16); i++) {  // 16 keys: 8 columns of fp16 pairs; low parts first
                    const int ks = i % (TR_KB / 16);
                    umma_f16_tmem(d, p + (i < TR_KB / 16 ? 32 : 0) + 8 * ks, vd + ks * (2048 >> 4), IDESC_O,
                                  i > 0 ? 1u : 0u);
                }
                umma_commit(&o_done[0][c & 1]);
                umma_commit(&v_empty[st]);
                return true;
            };
            do {
                const int nb = w.blk1 - w.blk0;
                ok = tr_wait(&q_full, (uint32_t)seg & 1u) && issue_s(j);
                if (ok && nb == 1) umma_commit(&q_empty);
                for (int k = 0; ok && k < nb && !s_abort; k++, j++) {
                    if (k + 1 < nb) {
                        ok = issue_s(j + 1);
                        if (k + 2 == nb) umma_commit(&q_empty);
                    }
                    ok = ok && issue_o(j);
                }
                seg++;
            } while (ok && !s_abort && w.next(A));
            if (!ok) s_abort = 1;
            umma_commit(&fin[0]);  // every MMA issued has completed before TMEM is released
            mbar_wait_bounded(&fin[0], 0);
        }
    } else if (!C::LO && (warp == 9 || warp == 11)) {
        // ---- MMA issue for group g: its next scores before its products of this block.  (The tensor core runs one
        // thread's products in order: a score buffer is rewritten after the product that read it.)
        if (lane == 0) {
            const int g = warp == 11;
            // descriptors advance by adding to their address field (16-byte units)
            const uint64_t dQ = umma_desc_sw128(smem_u32(sQ)), dV = umma_desc_mn_sw128(smem_u32(sV), TR_KB * 128, 1024);
            const uint64_t dK = PAGE == 64 ? umma_desc_mn_sw128(smem_u32(sK), C::KV_BYTES, 1024)
                                           : umma_desc_mn_sw64(smem_u32(sK), HD * PAGE * 2, 512);
            const uint32_t t_s = tmem + 128 * g, t_o = tmem + TR_O_COL + HD * g;
            int cb = 0, jb = 0, seg = 0;  // blocks and jobs of the segments before this one
            bool ok = true;
            do {
                const bool both = w.both();
                const int nj = w.jobs(g), step = both ? 1 : 2;
                const uint64_t dq = dQ + (both ? g : 0) * (C::TILE_BYTES >> 4);
                // the next blocks' full barriers and phases
                const int c0 = cb + (both ? 0 : g);
                int kf = c0 % (2 * ST), vf = kf;
                uint32_t kph = (uint32_t)(c0 / (2 * ST)) & 1u, vph = kph;
                auto forward = [&](int &f, uint32_t &ph) {
                    f += step;
                    if (f >= 2 * ST) {
                        f -= 2 * ST;
                        ph ^= 1;
                    }
                };
                // a stage is free once both groups are done with it, or with one tile the block's only one
                auto release = [&](uint64_t *bar) {
                    umma_commit(bar);
                    if (!both) mbar_arrive(bar);
                };
                auto issue_s = [&](int k) -> bool {
                    const int j = jb + k;
                    const uint32_t d = t_s + TR_KB * (j & 1);
                    const int st = kf >= ST ? kf - ST : kf;
                    const uint64_t kd = dK + st * (C::KV_BYTES >> 4);
                    if (!tr_wait(&k_full[kf], kph)) return false;
                    tc_fence_after();
#pragma unroll
                    for (int ks = 0; ks < HD / 16; ks++) {  // 16 dims: 16 rows of the dim-major pages
                        const uint32_t qo = ((uint32_t)(ks >> 2) * (TR_ROWS * 128) + (uint32_t)(ks & 3) * 32) >> 4;
                        umma_f16_desc(d, dq + qo, kd + ks * (16 * PAGE * 2 >> 4), IDESC_S, ks > 0 ? 1u : 0u);
                    }
                    umma_commit(&s_full[g][j & 1]);
                    release(&k_empty[st]);
                    forward(kf, kph);
                    if (k + 1 == nj) umma_commit(&q_empty);
                    return true;
                };
                auto issue_o = [&](int k) -> bool {
                    const int j = jb + k;
                    const uint32_t p = t_s + TR_KB * (j & 1);
                    const int st = vf >= ST ? vf - ST : vf;
                    const uint64_t vd = dV + st * (C::KV_BYTES >> 4);
                    if (!tr_wait(&v_full[vf], vph)) return false;
                    if (k == 0 && seg > 0 && !tr_wait(&o_free, (uint32_t)(seg - 1) & 1u)) return false;
                    if (!tr_wait(&p_full[g][j & 1], (uint32_t)(j >> 1) & 1u)) return false;
                    tc_fence_after();
#pragma unroll
                    for (int i = 0; i < (C::PLO ? 2 : 1) * (TR_KB / 16); i++) {  // 16 keys: 8 columns of fp16 pairs
                        const int ks = i % (TR_KB / 16);
                        const uint32_t part = C::PLO && i < TR_KB / 16 ? 32 : 0;  // the low parts first
                        umma_f16_tmem(t_o, p + part + 8 * ks, vd + ks * (2048 >> 4), IDESC_O, (k > 0 || i > 0) ? 1u : 0u);
                    }
                    umma_commit(&o_done[g][j & 1]);
                    release(&v_empty[st]);
                    forward(vf, vph);
                    return true;
                };
                ok = tr_wait(&q_full, (uint32_t)seg & 1u);
                if (ok && nj == 0) mbar_arrive(&q_empty);
                if (ok && nj > 0) ok = issue_s(0);
                for (int k = 0; ok && k < nj && !s_abort; k++) ok = (k + 1 >= nj || issue_s(k + 1)) && issue_o(k);
                cb += w.blk1 - w.blk0;
                jb += nj;
                seg++;
            } while (ok && !s_abort && w.next(A));
            if (!ok) s_abort = 1;
            umma_commit(&fin[g]);  // every MMA issued has completed before TMEM is released
            mbar_wait_bounded(&fin[g], 0);
        }
    } else {
        // ---- softmax: group g, thread = row r of its tile (TMEM lane)
        constexpr unsigned FULL = 0xffffffffu;
        const int qd = warp & 3, g = warp >> 2, r = 32 * qd + lane;
        const uint32_t lt = tmem + ((uint32_t)(32 * qd) << 16);
        const uint32_t t_s = lt + 128 * g, t_o = lt + TR_O_COL + HD * g;
        const float sign = A.scale < 0.f ? -1.f : 1.f;
        uint32_t npair = 0;  // uses of pair_bar[qd]
        bool ok = true;
        int cb = 0, jb = 0, seg = 0;  // blocks and this group's jobs of the segments before
        // The group's queries as fp16 parts scaled by 2^-e: HD / 8 lanes a row, the first 8 (or 4) warps share the
        // rows.  f32: batches of eight loads through registers.  16-bit: copied as they are into their places, all
        // copies in flight together, and (bf16) turned in place by the thread that copied them, in rolled loops: code
        // that runs once a segment arrives more slowly than it executes.
        auto load_q = [&](const TreeWalk &t, int sg, int warps) {
            constexpr int LPR = HD / 8, RPI = 32 / LPR;
            const int rows = t.rows(A), each = (t.both() ? TR_PAIR : TR_ROWS) / warps, d = (lane % LPR) * 8;
            const T *base = static_cast<const T *>(A.q) + (int64_t)t.s.off * A.qt + (int64_t)t.h * A.group * HD + d;
            auto place = [&](int rr) {
                return sQ + (rr >> 7) * C::TILE_BYTES + (uint32_t)(d >> 6) * (TR_ROWS * 128) +
                       sw128_off(rr & 127, (d >> 3) & 7);
            };
            auto source = [&](int rr) {
                const int row = t.row0(A) + rr, tok = tree_token(A, row);
                return base + (int64_t)tok * A.qt + (int64_t)(row - tok * A.group) * HD;
            };
            auto turn = [&](float (&x)[8], int rr, uint4 &hi, uint4 &lo) {
                float mx = 0.f;
#pragma unroll
                for (int e = 0; e < 8; e++) mx = fmaxf(mx, fabsf(x[e]));
#pragma unroll
                for (int o = 1; o < LPR; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, o));
                const int ex = (int)((__float_as_uint(mx) >> 23) & 255u);
                const float f = __fmul_rn(sign, __uint_as_float((uint32_t)(127 - tree_shift(ex)) << 23));
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = __fmul_rn(x[e], f);
                split8(x, hi, lo);
                if (d == 0) s_qe[sg & 1][rr] = (uint8_t)ex;
            };
            if constexpr (C::LO) {
                constexpr int AHEAD = 8;
                for (int i0 = 0; i0 < each; i0 += RPI * AHEAD) {
                    float x[AHEAD][8];
#pragma unroll
                    for (int k = 0; k < AHEAD; k++) {
                        const int rr = warp * each + i0 + k * RPI + lane / LPR;
#pragma unroll
                        for (int e = 0; e < 8; e++) x[k][e] = 0.f;
                        if (i0 + k * RPI < each && rr < rows) tr_load8(source(rr), A.qvec, x[k]);
                    }
#pragma unroll
                    for (int k = 0; k < AHEAD; k++) {
                        if (i0 + k * RPI >= each) break;
                        const int rr = warp * each + i0 + k * RPI + lane / LPR;
                        uint4 hi, lo;
                        turn(x[k], rr, hi, lo);
                        *reinterpret_cast<uint4 *>(place(rr)) = hi;
                        *reinterpret_cast<uint4 *>(place(rr) + C::Q_BYTES) = lo;
                    }
                }
            } else {
#pragma unroll 1
                for (int i0 = 0; i0 < each; i0 += RPI) {
                    const int rr = warp * each + i0 + lane / LPR;
                    uint8_t *dst = place(rr);
                    if (rr >= rows) {
                        *reinterpret_cast<uint4 *>(dst) = make_uint4(0, 0, 0, 0);
                    } else if (A.qvec) {
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(source(rr))
                                     : "memory");
                    } else {
                        const T *src = source(rr);
#pragma unroll
                        for (int i = 0; i < 8; i++) reinterpret_cast<T *>(dst)[i] = src[i];
                    }
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                constexpr bool half = std::is_same<T, __half>::value;  // (f16 queries enter as they are)
                if (!half || A.scale < 0.f)
#pragma unroll 2
                    for (int i0 = 0; i0 < each; i0 += RPI) {
                        const int rr = warp * each + i0 + lane / LPR;
                        uint4 *dst = reinterpret_cast<uint4 *>(place(rr));
                        if constexpr (half) {
                            const uint4 q = *dst;
                            constexpr uint32_t S = 0x80008000u;
                            *dst = make_uint4(q.x ^ S, q.y ^ S, q.z ^ S, q.w ^ S);
                        } else {
                            float x[8];
                            uint4 lo;
                            tr_load8(reinterpret_cast<const T *>(dst), true, x);
                            turn(x, rr, *dst, lo);
                        }
                    }
            }
            fence_proxy_async_smem();  // the tensor core reads them through the async proxy
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&q_full);
                if (warps == 4) mbar_arrive(&q_full);  // (8 arrivals)
                if (sg == 0) mbar_arrive(&go);
            }
        };
        // a row's score unit, |scale| log2(e) 2^e (not 0: masked scores stay -inf)
        auto unit_of = [&](int sg, int rr) {
            float u = __fmul_rn(fabsf(A.scale), 1.4426950408889634f);
            if constexpr (!std::is_same<T, __half>::value)
                u = __fmul_rn(u, __uint_as_float((uint32_t)(127 + tree_shift(s_qe[sg & 1][rr])) << 23));
            return fmaxf(u, 1e-37f);
        };
        // Values of block c that some row must not see: 0 * NaN would reach it.  Behind the last key and in skipped
        // pages all are zeroed; at new rows the non-finite ones, which the rows that see them get back at the end
        // (s_odd).  By the 128 threads of a softmax group.  (With two tiles both groups do it, each before its own
        // product: they write the same values, and the flag before them.)
        auto mend_values = [&](const TreeWalk &t, int c, int p0, int skip, int sg) -> bool {
            const int st = c % ST, pre = t.s.len - t.s.n;
            if (!tr_wait(&v_full[c % (2 * ST)], (uint32_t)(c / (2 * ST)) & 1u)) return false;
            for (int i = threadIdx.x & 127; i < (int)C::KV_BYTES / 16; i += 128) {
                const int k = (i >> 3) & 63;
                uint4 *cell = reinterpret_cast<uint4 *>(sV + st * C::KV_BYTES) + i;
                if (p0 + k >= t.s.len || ((skip >> (k >> 5)) & 1)) {
                    *cell = make_uint4(0, 0, 0, 0);
                } else if (p0 + k >= pre) {
                    uint4 v = *cell;
                    uint32_t *e = reinterpret_cast<uint32_t *>(&v);
                    bool odd = false;
#pragma unroll
                    for (int i4 = 0; i4 < 4; i4++) {
                        if ((e[i4] & 0x7C00u) == 0x7C00u) {
                            e[i4] &= 0xffff0000u;
                            odd = true;
                        }
                        if ((e[i4] & 0x7C000000u) == 0x7C000000u) {
                            e[i4] &= 0xffffu;
                            odd = true;
                        }
                    }
                    if (odd) {
                        s_odd[sg & 1] = sg + 1;
                        __threadfence_block();
                        *cell = v;
                    }
                }
            }
            fence_proxy_async_smem();
            return true;
        };
        // What a row gets back of the non-finite values it sees: dimensions d0 .. d0 + 31.
        auto give_back = [&](const TreeWalk &t, int tok, int d0, float (&o)[32]) {
            const int pre = t.s.len - t.s.n;
            for (int i = max(0, t.blk0 * TR_KB - pre); i < min(t.s.n, t.blk1 * TR_KB - pre); i++) {
                const int p = pre + i, page = A.bt[(int64_t)t.b * A.max_pages + p / PAGE];
                if (page < 0 || page >= A.num_pages || !(tree_visible(A, t.s, tok, p) & 1)) continue;
                const __half *v = A.vpool + (((int64_t)page * A.n_kv + t.h) * PAGE + p % PAGE) * HD + d0;
#pragma unroll
                for (int e = 0; e < 32; e++) {
                    const float x = __half2float(v[e]);
                    if (!isfinite(x)) o[e] = __fadd_rn(o[e], x);
                }
            }
        };
        auto hide = [&](const TreeWalk &t, int tok, int p0, int skip, uint32_t (&sv)[64]) {  // scores of unseen keys
            const uint32_t v0 = skip & 1 ? 0u : tree_visible(A, t.s, tok, p0);
            const uint32_t v1 = skip & 2 ? 0u : tree_visible(A, t.s, tok, p0 + 32);
#pragma unroll
            for (int i = 0; i < 32; i++) {
                if (!((v0 >> i) & 1)) sv[i] = 0xff800000u;  // -inf
                if (!((v1 >> i) & 1)) sv[32 + i] = 0xff800000u;
            }
        };
        auto largest = [&](const uint32_t (&sv)[64]) {
            float b4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int t = 0; t < 64; t++) b4[t & 3] = fmaxf(b4[t & 3], __uint_as_float(sv[t]));
            return fmaxf(fmaxf(b4[0], b4[1]), fmaxf(b4[2], b4[3]));
        };
        // p = 2^(s u - m + 7) as fp16 pairs over the scores, low parts (not bf16) behind the high ones; their sum
        auto exponentials = [&](const uint32_t (&sv)[64], float u, float m, uint32_t t_b) {
            const float ref = __fsub_rn(TR_LIFT, m);
            float l4[4] = {0.f, 0.f, 0.f, 0.f};
            uint32_t hi[32], lo[32];
#pragma unroll
            for (int t = 0; t < 32; t++) {
                const float pa = exp2_approx(__fmaf_rn(__uint_as_float(sv[2 * t]), u, ref));
                const float pb = exp2_approx(__fmaf_rn(__uint_as_float(sv[2 * t + 1]), u, ref));
                const __half2 h2 = __floats2half2_rn(pa, pb);
                hi[t] = *reinterpret_cast<const uint32_t *>(&h2);
                l4[t & 3] = __fadd_rn(l4[t & 3], __fadd_rn(pa, pb));
                if (C::PLO) {
                    const float2 hf = __half22float2(h2);
                    const __half2 q2 = __floats2half2_rn(__fsub_rn(pa, hf.x), __fsub_rn(pb, hf.y));
                    lo[t] = *reinterpret_cast<const uint32_t *>(&q2);
                }
            }
            tmem_st32(t_b, hi);
            if (C::PLO) tmem_st32(t_b + 32, lo);
            return __fadd_rn(__fadd_rn(l4[0], l4[1]), __fadd_rn(l4[2], l4[3]));
        };
        // The maximum m is rounded down, and what a score exceeds it by is computed exactly; where f32 has no fractions
        // left at m's size that excess could reach 2^9 and more.  So far maxima are taken off first (s u - m, at most 8:
        // 2^15), and the exponentials see scores next to 0.
        auto far = [&](float m) { return __any_sync(FULL, fabsf(m) > TR_FAR && m != TR_NONE); };
        auto bring_near = [&](uint32_t (&sv)[64], float u, float m) {
#pragma unroll
            for (int t = 0; t < 64; t++) {
                const float x = __fmaf_rn(__uint_as_float(sv[t]), u, -m);
                sv[t] = __float_as_uint(x > 8.f ? 8.f : x);  // (NaN stays)
            }
        };
        if constexpr (C::LO) {
            // ---- f32: group 0 turns scores into probabilities, group 1 sums the blocks' products in registers
            load_q(w, 0, 8);
            if (g == 0) {
                for (;; seg++) {
                    const int nb = w.blk1 - w.blk0, pre = w.s.len - w.s.n, rows = w.rows(A);
                    const bool active = rows > 32 * qd;
                    const int row = w.row0(A) + min(r, rows - 1), tok = tree_token(A, row);
                    if (!(ok = tr_wait(&q_full, (uint32_t)seg & 1u))) break;
                    // (what segment seg - 2 left for group 1 has been taken)
                    if (seg >= 2 && !(ok = tr_wait(&ml_read[seg & 1], (uint32_t)((seg >> 1) - 1) & 1u))) break;
                    const float u = unit_of(seg, r);
                    float m = TR_NONE, l = 0.f;
                    for (int k = 0; k < nb; k++) {
                        const int j = jb + k, p0 = (w.blk0 + k) * TR_KB;
                        const uint32_t t_b = lt + TR_KB * (j & 1);
                        if (!(ok = tr_wait(&s_full[0][j & 1], (uint32_t)(j >> 1) & 1u))) break;
                        tc_fence_after();
                        const int skip = s_skip[j & 15];
                        const bool odd = p0 + TR_KB > pre || skip;
                        if (active) {
                            uint32_t sv[64];
                            tmem_ld64(t_b, sv);
                            if (odd) hide(w, tok, p0, skip, sv);
                            const float mn = fmaxf(m, __fmul_rd(largest(sv), u));
                            const float al = exp2f(__fsub_rn(m, mn));
                            m = mn;
                            // (four blocks in flight at most: the product of block j - 2 waits for the reader of j - 4)
                            s_al[j & 3][r] = al;
                            float sum;
                            if (__builtin_expect(far(m), 0)) {
                                bring_near(sv, u, m);
                                sum = exponentials(sv, 1.f, 0.f, t_b);
                            } else {
                                sum = exponentials(sv, u, m, t_b);
                            }
                            l = __fmaf_rn(l, al, sum);
                        }
                        if (odd && !(ok = mend_values(w, j, p0, skip, seg))) break;
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&p_full[0][j & 1]);
                    }
                    if (!ok) break;
                    s_ml[seg & 1][r] = make_float2(m, l);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&ml_full[seg & 1]);
                    jb += nb;
                    // the next segment's queries, once this one's last scores are out
                    if (!w.next(A) || !(ok = tr_wait(&q_empty, (uint32_t)seg & 1u))) break;
                    load_q(w, seg + 1, 4);
                }
            } else {
                float acc[HD];
                for (;; seg++) {
                    const int nb = w.blk1 - w.blk0, rows = w.rows(A);
                    const bool active = rows > 32 * qd;
                    const int row = w.row0(A) + min(r, rows - 1), tok = tree_token(A, row);
#pragma unroll
                    for (int e = 0; e < HD; e++) acc[e] = 0.f;
                    for (int k = 0; k < nb; k++) {
                        const int j = jb + k;
                        if (!(ok = tr_wait(&o_done[0][j & 1], (uint32_t)(j >> 1) & 1u))) break;
                        tc_fence_after();
                        if (active) {
                            const float al = s_al[j & 3][r];
#pragma unroll
                            for (int i = 0; i < HD / 16; i++) {
                                uint32_t ov[16];
                                tmem_ld16(lt + TR_O_COL + HD * (j & 1) + 16 * i, ov);
#pragma unroll
                                for (int e = 0; e < 16; e++)
                                    acc[16 * i + e] = __fmaf_rn(acc[16 * i + e], al, __uint_as_float(ov[e]));
                            }
                        }
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&o_read[j & 1]);
                    }
                    if (!ok) break;
                    jb += nb;
                    // ---- this segment's rows
                    if (!(ok = tr_wait(&ml_full[seg & 1], (uint32_t)(seg >> 1) & 1u))) break;
                    const float2 ml = s_ml[seg & 1][r];
                    const bool odd = s_odd[seg & 1] == seg + 1, whole = !A.split || w.whole();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&ml_read[seg & 1]);
                    const float inv = ml.y > 0.f ? __fdiv_rn(1.f, ml.y) : 0.f;
                    float *part = A.part + (int64_t)(2 * blockIdx.x + (w.blk0 == 0)) * (HD + 2) * A.rows_cap;
                    T *orow = static_cast<T *>(A.out) + (int64_t)(w.s.off + tok) * A.ot +
                              (int64_t)(w.h * A.group + row - tok * A.group) * HD;
                    if (active) {
#pragma unroll
                        for (int d0 = 0; d0 < HD; d0 += 32) {
                            float (&o)[32] = *reinterpret_cast<float (*)[32]>(&acc[d0]);
                            if (odd) give_back(w, tok, d0, o);
                            if (!whole) {
#pragma unroll
                                for (int i = 0; i < 32; i += 4)  // [dim / 4][row]: a warp stores 512 bytes at once
                                    reinterpret_cast<float4 *>(part)[(int64_t)((d0 + i) >> 2) * A.rows_cap + r] =
                                        make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                            } else if (r < rows) {
#pragma unroll
                                for (int i = 0; i < 32; i += 8) {
                                    float y[8];
#pragma unroll
                                    for (int e = 0; e < 8; e++) y[e] = __fmul_rn(o[i + e], inv);
                                    tr_store8(orow + d0 + i, A.ovec, y);
                                }
                            }
                        }
                        if (!whole) reinterpret_cast<float2 *>(part + (int64_t)HD * A.rows_cap)[r] = ml;
                    }
                    if (!w.next(A)) break;
                }
            }
        } else {
        // A pass: the next segment's queries go in once this one's last scores are out, then this one's rows are
        // written, then the next one's blocks.
        TreeWalk nw = w;
        bool first = true, more = true, active = false;
        int nj = 0, tile_rows = 0, row = 0, tok = 0;
        float m = TR_NONE, l = 0.f;
        for (;;) {
            if (more) {
                if (!first && !(ok = tr_wait(&q_empty, (uint32_t)seg & 1u))) break;
                load_q(nw, first ? 0 : seg + 1, 8);
            }
            if (!first) {
                const bool both = w.both();
                // ---- this segment's rows, once the last products have landed
                if (nj > 0) {
                    const int j = jb + nj - 1;
                    if (!(ok = tr_wait(&o_done[g][j & 1], (uint32_t)(j >> 1) & 1u))) break;
                }
                // One tile: group 0 takes over group 1's part (if that had a block) and writes the rows.
                const bool two = !both && w.jobs(1) > 0;
                float w0 = 1.f, w1 = 0.f;
                if (two) {
                    if (g == 1) {
                        s_ml[0][r] = make_float2(m, l);
                        tc_fence_before();
                        mbar_arrive(&pair_bar[qd]);
                    } else {
                        if (!(ok = tr_wait(&pair_bar[qd], npair & 1u))) break;
                        const float2 o = s_ml[0][r];
                        const float mm = fmaxf(m, o.x);
                        w0 = exp2f(__fsub_rn(m, mm));
                        w1 = exp2f(__fsub_rn(o.x, mm));
                        m = mm;
                        l = __fmaf_rn(w0, l, __fmul_rn(w1, o.y));
                    }
                    npair++;
                }
                tc_fence_after();
                if (active && (both || g == 0)) {
                    const bool odd = s_odd[seg & 1] == seg + 1, whole = !A.split || w.whole();
                    const float inv = l > 0.f ? __fdiv_rn(1.f, l) : 0.f;
                    const int pr = (both ? TR_ROWS * g : 0) + r;  // row of the partial
                    float *part = A.part + (int64_t)(2 * blockIdx.x + (w.blk0 == 0)) * (HD + 2) * A.rows_cap;
                    T *orow = static_cast<T *>(A.out) + (int64_t)(w.s.off + tok) * A.ot +
                              (int64_t)(w.h * A.group + row - tok * A.group) * HD;
#pragma unroll 1
                    for (int d0 = 0; d0 < HD; d0 += 32) {
                        uint32_t ov[32];
                        tmem_ld32(t_o + d0, ov);
                        if (two) {
                            uint32_t o1[32];
                            tmem_ld32(t_o + HD + d0, o1);
#pragma unroll
                            for (int i = 0; i < 32; i++)
                                ov[i] = __float_as_uint(
                                    __fmaf_rn(w1, __uint_as_float(o1[i]), __fmul_rn(w0, __uint_as_float(ov[i]))));
                        }
                        if (odd) {
                            float o[32];
#pragma unroll
                            for (int e = 0; e < 32; e++) o[e] = __uint_as_float(ov[e]);
                            give_back(w, tok, d0, o);
#pragma unroll
                            for (int e = 0; e < 32; e++) ov[e] = __float_as_uint(o[e]);
                        }
                        if (!whole) {
#pragma unroll
                            for (int i = 0; i < 32; i += 4)  // [dim / 4][row]: a warp stores 512 bytes at once
                                reinterpret_cast<uint4 *>(part)[(int64_t)((d0 + i) >> 2) * A.rows_cap + pr] =
                                    make_uint4(ov[i], ov[i + 1], ov[i + 2], ov[i + 3]);
                        } else if (r < tile_rows) {
#pragma unroll
                            for (int i = 0; i < 32; i += 8) {
                                float y[8];
#pragma unroll
                                for (int e = 0; e < 8; e++) y[e] = __fmul_rn(__uint_as_float(ov[i + e]), inv);
                                tr_store8(orow + d0 + i, A.ovec, y);
                            }
                        }
                    }
                    if (!whole)
                        reinterpret_cast<float2 *>(part + (int64_t)HD * A.rows_cap)[pr] = make_float2(m, l);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&o_free);
                cb += w.blk1 - w.blk0;
                jb += nj;
                seg++;
            }
            if (!more) break;
            first = false;
            w = nw;
            const bool both = w.both();
            const int pre = w.s.len - w.s.n;
            nj = w.jobs(g);
            tile_rows = w.rows(A) - (both ? TR_ROWS * g : 0);  // of this group's tile
            active = tile_rows > 32 * qd;
            row = w.row0(A) + (both ? TR_ROWS * g : 0) + min(r, tile_rows - 1);
            tok = tree_token(A, row);
            if (!(ok = tr_wait(&q_full, (uint32_t)seg & 1u))) break;
            const float sl2 = unit_of(seg, (both ? TR_ROWS * g : 0) + r);
            m = TR_NONE;
            l = 0.f;
            for (int k = 0; k < nj; k++) {
                const int j = jb + k, blk = w.blk0 + (both ? k : 2 * k + g), c = cb + (blk - w.blk0), p0 = blk * TR_KB;
                const uint32_t t_b = t_s + TR_KB * (j & 1);
                // (these scores were issued behind the group's product of job j - 2: that one has landed too, so of
                // the o_done phases only those of j - 1 and j can be open below)
                if (!(ok = tr_wait(&s_full[g][j & 1], (uint32_t)(j >> 1) & 1u))) break;
                tc_fence_after();
                const int skip = s_skip[c & 15];
                if (active) {
                    uint32_t sv[64];
                    tmem_ld64(t_b, sv);
                    if (p0 + TR_KB > pre || skip) hide(w, tok, p0, skip, sv);
                    const float bm = largest(sv);
                    const float mn = fmaxf(m, __fmul_rd(bm, sl2));
                    const bool need = k > 0 && mn > m + 8.f;
                    if (__any_sync(FULL, need)) {
                        // rescale the accumulator rows once the product of this group's last block has landed
                        if (!(ok = tr_wait(&o_done[g][(j - 1) & 1], (uint32_t)((j - 1) >> 1) & 1u))) break;
                        tc_fence_after();
                        const float al = need ? exp2_approx(__fsub_rn(m, mn)) : 1.f;
#pragma unroll 1
                        for (int i = 0; i < HD / 32; i++) {
                            uint32_t ov[32];
                            tmem_ld32(t_o + 32 * i, ov);
#pragma unroll
                            for (int e = 0; e < 32; e++) ov[e] = __float_as_uint(__fmul_rn(__uint_as_float(ov[e]), al));
                            tmem_st32(t_o + 32 * i, ov);
                        }
                        if (need) {
                            l = __fmul_rn(l, al);
                            m = mn;
                        }
                    }
                    if (k == 0) m = mn;
                    if (__builtin_expect(far(m), 0)) {
                        bring_near(sv, sl2, m);
                        l = __fadd_rn(l, exponentials(sv, 1.f, 0.f, t_b));
                    } else {
                        l = __fadd_rn(l, exponentials(sv, sl2, m, t_b));
                    }
                }
                if ((p0 + TR_KB > pre || skip) && !(ok = mend_values(w, c, p0, skip, seg))) break;
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[g][j & 1]);
            }
            if (!ok) break;
            more = nw.next(A);
        }
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

// Joins the partials of the row groups that several CTAs hold.  grid (row groups a
// kv head x rows_cap / 32 x HD / (16 COLS), n_kv, batch): a warp has eight rows by
// four COLS columns of four dimensions, so that it reads the parts by 128 bytes and
// writes whole 32-byte sectors of the rows (with a lane a row and single values the
// writes alone took 10 us of 16 sequences of 25 tokens, 32 heads); the loads of
// eight (part, column) pairs are in flight together.  Finding a group's parts costs
// a block more than reading them, so where there are blocks enough a lane takes
// four columns, which saves 3 us of those sequences' call (8.5 us cold, 12.5 before).
template <typename T, int HD, int COLS>
__global__ void __launch_bounds__(128) k_attn_tree_join(const __grid_constant__ TreeArgs A) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int CG = HD / (16 * COLS), JOIN = 8 / COLS;  // column groups; parts whose loads are in flight together
    const int cgroup = blockIdx.x % CG, rest = blockIdx.x / CG;
    const int slabs = A.rows_cap / 32, slab = rest % slabs, pair = rest / slabs;
    const int b = blockIdx.z;
    TreeSeq s;
    s.load(A, b);
    const int row0 = pair * A.grows + 32 * slab;
    // (a block without work waits too: what is behind this kernel on the stream waits for it alone, so it must not end
    // before the attention has)
    if (row0 >= s.n * A.group) {
        pdl_wait();
        return;
    }
    // units before this sequence, and in all
    TreeTotal t{}, before{};
    for (int i = lane; i < A.batch; i += 32) {
        TreeSeq o;
        o.load(A, i);
        t.add(A, o);
        if (i < b) before.add(A, o);
    }
    t.reduce();
    before.reduce();
    const int quota = t.quota(A), lead = t.lead(A);
    const int wt = pair < s.pairs - 1 ? s.full : s.weight;
    // the group's first block's first unit
    const int gs = before.units + before.groups * lead + blockIdx.y * s.head_units(A, lead) +
                   pair * (s.full * s.blocks + lead) + lead;
    const int c0 = gs / quota, c1 = (gs + wt * (s.blocks - 1)) / quota;          // CTAs of its first and last block
    if (c0 == c1) {  // written by its CTA
        pdl_wait();
        return;
    }
    const int rr = row0 + 8 * warp + (lane & 7), r = rr - pair * A.grows;
    const int64_t slot = (int64_t)(HD + 2) * A.rows_cap;
    // the CTA with the group's first block keeps it as its partial 1, the others as their 0
    auto part = [&](int c) { return A.part + (2 * (int64_t)c + (c == c0)) * slot; };
    pdl_wait();
    const int col = cgroup * 4 * COLS + (lane >> 3);  // and every 4th from there
    float M = TR_NONE, L = 0.f;
    float4 o[COLS];
#pragma unroll
    for (int k = 0; k < COLS; k++) o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = c0; c <= c1; c += JOIN) {
        float2 ml[JOIN];
        float4 v[JOIN][COLS];
#pragma unroll
        for (int i = 0; i < JOIN; i++)
            if (c + i <= c1) {
                const float *p = part(c + i);
                ml[i] = reinterpret_cast<const float2 *>(p + (int64_t)HD * A.rows_cap)[r];
#pragma unroll
                for (int k = 0; k < COLS; k++)
                    v[i][k] = reinterpret_cast<const float4 *>(p)[(int64_t)(col + 4 * k) * A.rows_cap + r];
            }
        float mn = M;
#pragma unroll
        for (int i = 0; i < JOIN; i++)
            if (c + i <= c1) mn = fmaxf(mn, ml[i].x);
        const float al = exp2f(__fsub_rn(M, mn));  // (1 where nothing has been seen yet: there is nothing to scale)
        M = mn;
        L = __fmul_rn(L, al);
#pragma unroll
        for (int k = 0; k < COLS; k++)
            o[k] = make_float4(__fmul_rn(o[k].x, al), __fmul_rn(o[k].y, al), __fmul_rn(o[k].z, al),
                               __fmul_rn(o[k].w, al));
#pragma unroll
        for (int i = 0; i < JOIN; i++)
            if (c + i <= c1) {
                const float wgt = exp2f(__fsub_rn(ml[i].x, M));
                L = __fmaf_rn(wgt, ml[i].y, L);
#pragma unroll
                for (int k = 0; k < COLS; k++) {
                    o[k].x = __fmaf_rn(wgt, v[i][k].x, o[k].x);
                    o[k].y = __fmaf_rn(wgt, v[i][k].y, o[k].y);
                    o[k].z = __fmaf_rn(wgt, v[i][k].z, o[k].z);
                    o[k].w = __fmaf_rn(wgt, v[i][k].w, o[k].w);
                }
            }
    }
    if (rr >= s.n * A.group) return;
    const float inv = L > 0.f ? __fdiv_rn(1.f, L) : 0.f;
    const int tok = tree_token(A, rr);
    T *out = static_cast<T *>(A.out) + (int64_t)(s.off + tok) * A.ot +
             (int64_t)(blockIdx.y * A.group + rr - tok * A.group) * HD + 4 * col;
#pragma unroll
    for (int k = 0; k < COLS; k++) {
        alignas(16) T y[4];
        tr_put(y, __fmul_rn(o[k].x, inv));
        tr_put(y + 1, __fmul_rn(o[k].y, inv));
        tr_put(y + 2, __fmul_rn(o[k].z, inv));
        tr_put(y + 3, __fmul_rn(o[k].w, inv));
        if (A.ovec) {
            using W = typename std::conditional<sizeof(T) == 4, uint4, uint2>::type;
            *reinterpret_cast<W *>(out + 16 * k) = *reinterpret_cast<const W *>(y);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) out[16 * k + i] = y[i];
        }
    }
}

// What a call of these sizes launches.
struct TreePlan {
    int split, ctas, rows_cap, pairs;
    int64_t ws;
};
static TreePlan tree_plan(const fb_ctx *ctx, int batch, int max_new, int n_heads, int n_kv, int head_dim,
                          int max_seq_len, int grows) {
    TreePlan p{};
    const int64_t rows = (int64_t)max_new * (n_heads / n_kv);
    const int64_t pairs = (rows + grows - 1) / grows, blocks = (max_seq_len + TR_KB - 1) / TR_KB;
    const int64_t groups = pairs * n_kv * batch;
    FB_REQUIRE(groups * (2 * blocks + TR_SWITCH) < ((int64_t)1 << 31) - 4096 && pairs <= 65535,
               "attn_tree: batch too large");
    FB_REQUIRE((rows + TR_PAIR) * (n_heads / n_kv) < ((int64_t)1 << 32), "attn_tree: too many rows");
    p.split = blocks > TR_WHOLE;
    const int64_t units = 2 * groups * (p.split ? blocks : 1);
    p.ctas = (int)(units < ctx->num_sms ? units : ctx->num_sms);
    p.pairs = (int)pairs;
    p.rows_cap = (int)(rows >= grows ? grows : (rows + 31) / 32 * 32);
    p.ws = p.split ? (int64_t)2 * p.ctas * (head_dim + 2) * p.rows_cap * 4 : 0;
    return p;
}

template <typename T, int HD, int PAGE>
static void launch_tree(fb_ctx *ctx, const TreeArgs &A, const TreePlan &plan, const CUtensorMap &kmap,
                        const CUtensorMap &vmap) {
    constexpr size_t smem = TreeCfg<T, HD>::SMEM;
    FB_CUDA(cudaFuncSetAttribute(k_attn_tree<T, HD, PAGE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    launch_with(ctx->stream, ctx->pdl, k_attn_tree<T, HD, PAGE>, dim3((unsigned)plan.ctas), TR_THREADS, smem, 1, kmap,
               vmap, A);
    if (!plan.split) return;
    // the join's blocks start while the attention drains and wait for it
    const int64_t slabs = (int64_t)plan.pairs * (plan.rows_cap / 32);
    auto join = [&](auto kernel, int cols) {
        launch_with(ctx->stream, ctx->pdl, kernel,
                    dim3((unsigned)(slabs * (HD / (16 * cols))), (unsigned)A.n_kv, (unsigned)A.batch), 128, 0, 1, A);
    };
    if (slabs * (HD / 64) * A.n_kv * A.batch >= 4 * ctx->num_sms) join(k_attn_tree_join<T, HD, 4>, 4);
    else join(k_attn_tree_join<T, HD, 1>, 1);
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
        *bytes = 0;
        if (batch && max_new && max_seq_len)  // (of any dtype)
            for (int grows : {TR_ROWS, TR_PAIR}) {
                const int64_t ws =
                    tree_plan(ctx, batch, max_new, n_heads, n_kv_heads, head_dim, max_seq_len, grows).ws;
                *bytes = ws > *bytes ? ws : *bytes;
            }
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
        FB_REQUIRE(!rows_overlap(q_dev, q_token_stride, 0, out_dev, out_token_stride, 0, n_rows, 1,
                                 (int64_t)n_heads * head_dim, esz),
                   "attn_tree: q and out must not overlap");
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
        const int grows = dtype == FB_F32 ? TR_ROWS : TR_PAIR;
        const TreePlan plan = tree_plan(ctx, batch, max_new, n_heads, n_kv_heads, head_dim, max_seq_len, grows);
        FB_REQUIRE(plan.ws == 0 || (workspace_dev && workspace_bytes >= plan.ws && ((uintptr_t)workspace_dev & 15) == 0),
                   "attn_tree: the workspace must be 16-byte aligned and hold fb_attn_tree_workspace bytes (" +
                       std::to_string(plan.ws) + ")");
        A.group = n_heads / n_kv_heads;
        A.inv_group = (((uint64_t)1 << 32) + A.group - 1) / A.group;
        A.split = plan.split;
        A.ctas = plan.ctas;
        A.grows = grows;
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
