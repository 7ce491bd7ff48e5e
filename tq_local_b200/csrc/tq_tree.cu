// Attention of drafted tokens over the packed cache.  The T drafted tokens of every batch entry are packed at tokens
// [tree_start, tree_start + T); node i attends the entry's history [seq_start, length) and the drafted tokens that its mask names:
//
//   logit_ij = scale (kn_j c_k[codes_j] . (R_k q_i) + rn_j sqrt(pi/2)/D signs_j . (S q_i)),   out_i = R_v^T sum_j p_ij vn_j c_v[codes_j]
//
// One warp per (node, head): a pass over its tokens with the running maximum and sum of the softmax, four coordinates a lane.
#include <math.h>

#include "tq_common.cuh"

namespace {

struct TreeArgs {
    const uint8_t *k_codes, *k_signs, *v_codes;
    const uint16_t *k_norms, *k_rnorms, *v_norms;
    int64_t cache_sb, cache_sh;
    int key_bits, bits, use_qjl, kv_heads, group, nodes, tree_start;
    const int *seq_start, *lengths;
    const uint64_t *mask;
    const float *rot_k_t, *rot_v, *qjl_t, *centers_k, *centers_v;
    const void *q;
    void *out;
    int64_t qb, qh, qt, ob, oh, ot;
};

__device__ __forceinline__ int code_at(const uint8_t *p, int bits, int e) {
    const int bit = e * bits, byte = bit >> 3, sh = bit & 7;
    int w = p[byte];
    if (sh + bits > 8) w |= p[byte + 1] << 8;
    return (w >> sh) & ((1 << bits) - 1);
}

template <typename T> __global__ void __launch_bounds__(128) tq_tree_kernel(const __grid_constant__ TreeArgs a) {
    __shared__ float s_vec[4][TQ_D];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, i = blockIdx.x * 4 + w, hq = blockIdx.y, b = blockIdx.z;
    if (i >= a.nodes) return;
    const T *q = reinterpret_cast<const T *>(a.q) + b * a.qb + hq * a.qh + i * a.qt;
    for (int e = 0; e < 4; ++e) s_vec[w][4 * lane + e] = tq_to_float<T>(q[4 * lane + e]);
    __syncwarp();
    float qr[4] = {}, qp[4] = {};
    for (int d = 0; d < TQ_D; ++d)
        for (int e = 0; e < 4; ++e) {
            qr[e] += a.rot_k_t[d * TQ_D + 4 * lane + e] * s_vec[w][d];
            if (a.use_qjl) qp[e] += a.qjl_t[d * TQ_D + 4 * lane + e] * s_vec[w][d];
        }
    const int64_t row = b * a.cache_sb + hq / a.group * a.cache_sh;
    const int first = a.seq_start ? max(a.seq_start[b], 0) : 0;
    const int length = a.lengths ? min(max(a.lengths[b], 0), a.tree_start) : a.tree_start;
    const uint64_t seen = a.mask ? a.mask[(int64_t)b * a.nodes + i] : 0;
    float m = -INFINITY, l = 0.f, o[4] = {};
    const float scale = 0.08838834764831845f, sketch = 1.2533141373155003f / (float)TQ_D;
    for (int j = min(first, length); j < length + a.nodes; ++j) {
        const int node = j - length;
        if (node >= 0 && !(a.mask ? seen >> node & 1 : node <= i)) continue;
        const int64_t t = row + (node < 0 ? j : a.tree_start + node);
        float s = 0.f, x = 0.f;
        for (int e = 0; e < 4; ++e) {
            s += qr[e] * a.centers_k[code_at(a.k_codes + t * 16 * a.key_bits, a.key_bits, 4 * lane + e)];
            if (a.use_qjl) x += code_at(a.k_signs + t * 16, 1, 4 * lane + e) ? qp[e] : -qp[e];
        }
        s *= tq_half_bits_to_float(a.k_norms[t]);
        if (a.use_qjl) s += x * sketch * tq_half_bits_to_float(a.k_rnorms[t]);
        s = scale * tq_warp_sum(s);
        const float m_new = fmaxf(m, s), keep = m_new == -INFINITY ? 1.f : expf(m - m_new), p = m_new == -INFINITY ? 0.f : expf(s - m_new);
        m = m_new, l = l * keep + p;
        const float pv = p * tq_half_bits_to_float(a.v_norms[t]);
        for (int e = 0; e < 4; ++e) o[e] = o[e] * keep + pv * a.centers_v[code_at(a.v_codes + t * 16 * a.bits, a.bits, 4 * lane + e)];
    }
    const float inv = l > 0.f || isnan(l) ? 1.f / l : 0.f;
    __syncwarp();
    for (int e = 0; e < 4; ++e) s_vec[w][4 * lane + e] = o[e] * inv;
    __syncwarp();
    float y[4] = {};
    for (int d = 0; d < TQ_D; ++d)
        for (int e = 0; e < 4; ++e) y[e] += s_vec[w][d] * a.rot_v[d * TQ_D + 4 * lane + e];
    T *out = reinterpret_cast<T *>(a.out) + b * a.ob + hq * a.oh + i * a.ot;
    for (int e = 0; e < 4; ++e) out[4 * lane + e] = tq_from_float<T>(y[e]);
}

bool aligned(const tq_dense_desc *d) {
    return !(((uintptr_t)d->data | (uintptr_t)(2 * (d->stride_b | d->stride_h | d->stride_t))) & 15);
}

}  // namespace

extern "C" size_t tq_tree_workspace_bytes(tq_ctx *ctx, int32_t batch, int32_t q_heads, int32_t kv_heads, int32_t n_nodes, int32_t n_tokens) {
    return 0;
}

extern "C" int32_t tq_tree_attn(tq_ctx *ctx, const tq_dense_desc *q, int32_t q_heads, int32_t n_nodes, const tq_cache_desc *cache,
                                int32_t tree_start, const int32_t *lengths, const uint64_t *tree_mask, void *workspace,
                                size_t workspace_bytes, const tq_dense_desc *out, tq_stream stream) {
    TqRange range_("tq_tree_attn");
    if (!ctx || !q || !out || !q->data || !out->data) return TQ_ERR_ARG;
    const int rc = tq_check_cache(ctx, cache);
    if (rc) return rc;
    if (q->dtype != TQ_DTYPE_F16 && q->dtype != TQ_DTYPE_BF16) return q->dtype == TQ_DTYPE_F32 ? TQ_ERR_UNSUPPORTED : TQ_ERR_ARG;
    if (out->dtype != q->dtype || !aligned(q) || !aligned(out)) return TQ_ERR_ARG;
    if (n_nodes < 0 || tree_start < 0 || (int64_t)tree_start + n_nodes > cache->capacity) return TQ_ERR_ARG;
    if (q_heads <= 0 || q_heads % cache->kv_heads) return TQ_ERR_ARG;
    if (q_heads / cache->kv_heads > TQ_MAX_GROUPS || (tree_mask && n_nodes > TQ_MAX_TREE)) return TQ_ERR_UNSUPPORTED;
    if (((uintptr_t)lengths & 3) || ((uintptr_t)tree_mask & 7)) return TQ_ERR_ARG;
    if (n_nodes == 0) return TQ_OK;
    TreeArgs a = {};
    a.k_codes = cache->k_codes, a.k_norms = cache->k_norms, a.k_signs = cache->k_signs, a.k_rnorms = cache->k_rnorms;
    a.v_codes = cache->v_codes, a.v_norms = cache->v_norms, a.cache_sb = cache->stride_b, a.cache_sh = cache->stride_h;
    a.key_bits = ctx->key_bits, a.bits = ctx->bits, a.use_qjl = ctx->use_qjl, a.kv_heads = cache->kv_heads;
    a.group = q_heads / cache->kv_heads, a.nodes = n_nodes, a.tree_start = tree_start;
    a.seq_start = cache->seq_start, a.lengths = lengths, a.mask = tree_mask;
    a.rot_k_t = ctx->rot_k_t, a.rot_v = ctx->rot_v, a.qjl_t = ctx->qjl_t, a.centers_k = ctx->centers_k, a.centers_v = ctx->centers_v;
    a.q = q->data, a.qb = q->stride_b, a.qh = q->stride_h, a.qt = q->stride_t;
    a.out = const_cast<void *>(out->data), a.ob = out->stride_b, a.oh = out->stride_h, a.ot = out->stride_t;
    const dim3 grid((n_nodes + 3) / 4, q_heads, cache->batch);
    if (q->dtype == TQ_DTYPE_F16) tq_tree_kernel<__half><<<grid, 128, 0, (cudaStream_t)stream>>>(a);
    else tq_tree_kernel<__nv_bfloat16><<<grid, 128, 0, (cudaStream_t)stream>>>(a);
    TQ_CUDA_CHECK(cudaGetLastError());
    return TQ_OK;
}
