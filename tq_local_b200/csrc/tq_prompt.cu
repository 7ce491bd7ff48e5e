// Attention of a whole prompt over dense keys and values: out_i = sum_j softmax_j(scale q_i . k_j) v_j over the keys a query sees.
//
// One warp per (query, head): a pass over its keys with the running maximum and sum of the softmax, four coordinates a lane.
#include <math.h>

#include "tq_common.cuh"

namespace {

__device__ int g_prompt_status;

struct PromptArgs {
    const void *q, *k, *v;
    void *out;
    int64_t qb, qh, qt, kb, kh, kt, vb, vh, vt, ob, oh, ot;
    int q_heads, group, n_q, n_kv;
    const int *seq_start, *cu_seqlens;
    float scale;
    bool causal;
};

template <typename T> __device__ __forceinline__ float4 load4(const void *base, int64_t at) {
    const T *p = reinterpret_cast<const T *>(base) + at;
    return make_float4(tq_to_float<T>(p[0]), tq_to_float<T>(p[1]), tq_to_float<T>(p[2]), tq_to_float<T>(p[3]));
}

template <typename T> __global__ void __launch_bounds__(128) tq_prompt_kernel(const __grid_constant__ PromptArgs a) {
    const int lane = threadIdx.x & 31, i = blockIdx.x * 4 + (threadIdx.x >> 5), h = blockIdx.y, b = blockIdx.z;
    int64_t t0 = 0;
    int n_q = a.n_q, n_kv = a.n_kv;
    if (a.cu_seqlens) t0 = a.cu_seqlens[b], n_q = n_kv = min(a.cu_seqlens[b + 1] - (int)t0, a.n_q);
    if (i >= n_q) return;
    const int64_t bb = a.cu_seqlens ? 0 : b;
    const float4 q = load4<T>(a.q, bb * a.qb + h * a.qh + (t0 + i) * a.qt + 4 * lane);
    const int first = a.seq_start ? max(a.seq_start[b], 0) : 0, last = a.causal ? min(n_kv, i + n_kv - n_q + 1) : n_kv;
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j = first; j < last; ++j) {
        const float4 k = load4<T>(a.k, bb * a.kb + h / a.group * a.kh + (t0 + j) * a.kt + 4 * lane);
        const float4 v = load4<T>(a.v, bb * a.vb + h / a.group * a.vh + (t0 + j) * a.vt + 4 * lane);
        const float s = a.scale * tq_warp_sum(q.x * k.x + q.y * k.y + q.z * k.z + q.w * k.w);
        const float m_new = fmaxf(m, s), keep = m_new == -INFINITY ? 1.f : expf(m - m_new), p = m_new == -INFINITY ? 0.f : expf(s - m_new);
        m = m_new, l = l * keep + p;
        o = make_float4(o.x * keep + p * v.x, o.y * keep + p * v.y, o.z * keep + p * v.z, o.w * keep + p * v.w);
    }
    const float inv = l > 0.f || isnan(l) ? 1.f / l : 0.f;
    T *p = reinterpret_cast<T *>(a.out) + bb * a.ob + h * a.oh + (t0 + i) * a.ot + 4 * lane;
    p[0] = tq_from_float<T>(o.x * inv), p[1] = tq_from_float<T>(o.y * inv), p[2] = tq_from_float<T>(o.z * inv), p[3] = tq_from_float<T>(o.w * inv);
}

bool aligned(const tq_dense_desc *d) {
    return !(((uintptr_t)d->data | (uintptr_t)(2 * (d->stride_b | d->stride_h | d->stride_t))) & 15);
}

int32_t prompt_attn(const tq_dense_desc *q, const tq_dense_desc *k, const tq_dense_desc *v, int32_t batch, int32_t q_heads,
                    int32_t kv_heads, int32_t n_q, int32_t n_kv, const int32_t *seq_start, const int32_t *cu_seqlens, float scale,
                    int32_t causal, void *workspace, size_t workspace_bytes, const tq_dense_desc *out, cudaStream_t stream) {
    if (!q || !k || !v || !out || !q->data || !k->data || !v->data || !out->data) return TQ_ERR_ARG;
    if (q->dtype != TQ_DTYPE_F16 && q->dtype != TQ_DTYPE_BF16) return q->dtype == TQ_DTYPE_F32 ? TQ_ERR_UNSUPPORTED : TQ_ERR_ARG;
    if (k->dtype != q->dtype || v->dtype != q->dtype || out->dtype != q->dtype) return TQ_ERR_ARG;
    if (batch < 0 || n_q < 0 || n_kv < 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads) return TQ_ERR_ARG;
    if (q_heads / kv_heads > TQ_MAX_PROMPT_GROUPS) return TQ_ERR_UNSUPPORTED;
    if (causal && n_kv < n_q) return TQ_ERR_ARG;
    if (!aligned(q) || !aligned(k) || !aligned(v) || !aligned(out)) return TQ_ERR_ARG;
    if (((uintptr_t)seq_start | (uintptr_t)cu_seqlens) & 3) return TQ_ERR_ARG;
    if (workspace_bytes < tq_prompt_workspace_bytes(batch, q_heads, kv_heads, n_q, n_kv)) return TQ_ERR_WORKSPACE;
    if (batch == 0 || n_q == 0) return TQ_OK;
    PromptArgs a = {};
    a.q = q->data, a.k = k->data, a.v = v->data, a.out = const_cast<void *>(out->data);
    a.qb = q->stride_b, a.qh = q->stride_h, a.qt = q->stride_t, a.kb = k->stride_b, a.kh = k->stride_h, a.kt = k->stride_t;
    a.vb = v->stride_b, a.vh = v->stride_h, a.vt = v->stride_t, a.ob = out->stride_b, a.oh = out->stride_h, a.ot = out->stride_t;
    a.q_heads = q_heads, a.group = q_heads / kv_heads, a.n_q = n_q, a.n_kv = n_kv, a.seq_start = seq_start, a.cu_seqlens = cu_seqlens;
    a.scale = scale, a.causal = causal != 0;
    const dim3 grid((n_q + 3) / 4, q_heads, batch);
    if (q->dtype == TQ_DTYPE_F16) tq_prompt_kernel<__half><<<grid, 128, 0, stream>>>(a);
    else tq_prompt_kernel<__nv_bfloat16><<<grid, 128, 0, stream>>>(a);
    TQ_CUDA_CHECK(cudaGetLastError());
    return TQ_OK;
}

}  // namespace

extern "C" size_t tq_prompt_workspace_bytes(int32_t batch, int32_t q_heads, int32_t kv_heads, int32_t n_q, int32_t n_kv) { return 0; }

extern "C" int32_t tq_prompt_attn(const tq_dense_desc *q, const tq_dense_desc *k, const tq_dense_desc *v, int32_t batch, int32_t q_heads,
                                  int32_t kv_heads, int32_t n_q, int32_t n_kv, const int32_t *seq_start, float scale, int32_t causal,
                                  void *workspace, size_t workspace_bytes, const tq_dense_desc *out, tq_stream stream) {
    TqRange range_("tq_prompt_attn");
    return prompt_attn(q, k, v, batch, q_heads, kv_heads, n_q, n_kv, seq_start, nullptr, scale, causal, workspace, workspace_bytes, out,
                       (cudaStream_t)stream);
}

extern "C" int32_t tq_prompt_attn_packed(const tq_dense_desc *q, const tq_dense_desc *k, const tq_dense_desc *v, int32_t n_seqs,
                                         int32_t total, int32_t q_heads, int32_t kv_heads, const int32_t *cu_seqlens, int32_t max_seqlen,
                                         float scale, int32_t causal, void *workspace, size_t workspace_bytes, const tq_dense_desc *out,
                                         tq_stream stream) {
    TqRange range_("tq_prompt_attn_packed");
    if (!cu_seqlens || total < 0 || max_seqlen < 0) return TQ_ERR_ARG;
    return prompt_attn(q, k, v, n_seqs, q_heads, kv_heads, max_seqlen, max_seqlen, nullptr, cu_seqlens, scale, causal, workspace,
                       workspace_bytes, out, (cudaStream_t)stream);
}

extern "C" int32_t tq_prompt_status(int32_t *status_out) {
    if (!status_out) return TQ_ERR_ARG;
    int v = 0;
    TQ_CUDA_CHECK(cudaMemcpyFromSymbol(&v, g_prompt_status, sizeof(v)));
    *status_out = v;
    return TQ_OK;
}
