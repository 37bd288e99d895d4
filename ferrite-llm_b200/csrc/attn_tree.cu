// Attention of drafted token trees over the paged cache (fb_attn_tree).  No
// reference counterpart: the reference verifies one chain, token by token
// (crates/ferrite-core/src/generation.rs:340-535).
//
// o = sum_j p_j v_j / sum_j p_j, p_j = exp(scale q.k_j - m), j over the prefix
// and the drafted tokens whose mask bit is set.
#include <math.h>

#include "fb_internal.h"
#include "kq_common.cuh"

namespace fb {

struct TreeArgs {
    const void *q;
    int64_t qt, ot;
    const __half *kpool, *vpool;
    const int32_t *bt, *offsets, *lens;
    const uint32_t *mask;
    int mask_words;
    void *out;
    int batch, n_rows, max_new, n_heads, n_kv, page, max_pages, num_pages, max_seq;
    float scale;
    uint32_t *err;
};

__device__ __forceinline__ float tr_f32(float v) { return v; }
__device__ __forceinline__ float tr_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float tr_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void tr_put(float *p, float v) { *p = v; }
__device__ __forceinline__ void tr_put(__half *p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void tr_put(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

// One warp per (new row, head): 32 keys a step, lane = key for the scores and
// lane = HD / 32 dimensions for the sums.
template <typename T, int HD>
__global__ void __launch_bounds__(128) k_attn_tree_simple(TreeArgs A) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int h = blockIdx.y * 4 + w, b = blockIdx.z;
    if (h >= A.n_heads) return;
    const int off = A.offsets[b], n = A.offsets[b + 1] - off, len = A.lens[b];
    if (off < 0 || n < 0 || n > A.max_new || off > A.n_rows - n || len < n || len > A.max_seq) {
        if (lane == 0) atomicOr(A.err, ERRBIT_BAD_POS);
        return;
    }
    const int i = blockIdx.x;
    if (i >= n) return;
    const int row = off + i, kvh = h / (A.n_heads / A.n_kv), pre = len - n;
    const T *q = static_cast<const T *>(A.q) + (int64_t)row * A.qt + (int64_t)h * HD;
    __shared__ float sq[4][HD];
    for (int d = lane; d < HD; d += 32) sq[w][d] = tr_f32(q[d]);
    __syncwarp();
    float m = -INFINITY, l = 0.f, o[HD / 32] = {};
    for (int p0 = 0; p0 < len; p0 += 32) {
        const int phys = A.bt[(int64_t)b * A.max_pages + p0 / A.page];
        if (phys < 0 || phys >= A.num_pages) {
            if (lane == 0) atomicOr(A.err, ERRBIT_BAD_PAGE);
            continue;
        }
        const int p = p0 + lane;
        bool see = p < len;
        if (see && p >= pre)
            see = A.mask ? (A.mask[(int64_t)row * A.mask_words + (p - pre) / 32] >> ((p - pre) % 32)) & 1 : p - pre <= i;
        const __half *k = A.kpool + ((int64_t)phys * A.n_kv + kvh) * HD * A.page + p % A.page;
        float s = -INFINITY;
        if (see) {
            s = 0.f;
            for (int d = 0; d < HD; d++) s = fmaf(sq[w][d], __half2float(k[(int64_t)d * A.page]), s);
            s *= A.scale;
        }
        float mn = s;
        for (int x = 16; x > 0; x >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, x));
        mn = fmaxf(m, mn);
        if (mn == -INFINITY && !__any_sync(0xffffffffu, see)) continue;
        const float al = m == -INFINITY ? 0.f : expf(m - mn), pr = see ? expf(s - mn) : 0.f;
        m = mn;
        float ps = pr;
        for (int x = 16; x > 0; x >>= 1) ps += __shfl_xor_sync(0xffffffffu, ps, x);
        l = l * al + ps;
        for (int e = 0; e < HD / 32; e++) o[e] *= al;
        const uint32_t seen = __ballot_sync(0xffffffffu, see);
        const __half *v = A.vpool + ((int64_t)phys * A.n_kv + kvh) * HD * A.page + (int64_t)(p0 % A.page) * HD;
        for (int t = 0; t < 32; t++) {
            const float pt = __shfl_sync(0xffffffffu, pr, t);
            if (!((seen >> t) & 1)) continue;
            for (int e = 0; e < HD / 32; e++) o[e] = fmaf(pt, __half2float(v[(int64_t)t * HD + lane + 32 * e]), o[e]);
        }
    }
    T *out = static_cast<T *>(A.out) + (int64_t)row * A.ot + (int64_t)h * HD;
    for (int e = 0; e < HD / 32; e++) tr_put(out + lane + 32 * e, l == 0.f ? 0.f : o[e] / l);
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
        A.page = page_size;
        A.max_pages = max_pages;
        A.num_pages = num_pages;
        A.max_seq = max_seq_len;
        A.scale = scale;
        A.err = ctx->err_word;
        const dim3 grid((unsigned)max_new, (unsigned)(n_heads + 3) / 4, (unsigned)batch);
        auto go = [&](auto t) {
            using T = decltype(t);
            if (head_dim == 128) k_attn_tree_simple<T, 128><<<grid, 128, 0, ctx->stream>>>(A);
            else k_attn_tree_simple<T, 64><<<grid, 128, 0, ctx->stream>>>(A);
        };
        if (dtype == FB_F32) go(float{});
        else if (dtype == FB_F16) go(__half{});
        else go(__nv_bfloat16{});
        FB_CUDA(cudaGetLastError());
    });
}

}  // extern "C"
