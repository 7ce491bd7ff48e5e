// Moves of packed tokens inside a cache, or from one cache to another: rows that become copies of other rows (beams that
// fork, requests that enter or leave a batch) and accepted drafted tokens that move behind their history.
//
// Both only carry bytes: six streams, in 16-byte units.  What bounds them is HBM for rows (16 rows of 8 heads x 32768 tokens, some of them copies of others,
// 457 MB read and written in place: 85 us, 5.4 TB/s or 0.82 of a plain copy's rate) and the launch for few of either (100 tokens of four rows 2.9 us,
// 12 accepted tokens 4.8, 64 of 64 sequences 5.8, each in a recorded graph).
#include "tq_common.cuh"

namespace {

constexpr int kStreams = 6;

struct Stream {
    const uint8_t *src;
    uint8_t *dst;
    int token_bytes;  // 16 x bits, 16 or 2
};

struct Streams {
    Stream s[kStreams];
    int n;
};

Streams streams_of(const tq_ctx *ctx, const tq_cache_desc *src, const tq_cache_desc *dst) {
    Streams r = {};
    auto add = [&](const void *from, void *to, int bytes) {
        r.s[r.n++] = {static_cast<const uint8_t *>(from), static_cast<uint8_t *>(to), bytes};
    };
    add(src->k_codes, dst->k_codes, 16 * ctx->key_bits);
    add(src->v_codes, dst->v_codes, 16 * ctx->bits);
    if (ctx->use_qjl) add(src->k_signs, dst->k_signs, 16);
    add(src->k_norms, dst->k_norms, 2);
    add(src->v_norms, dst->v_norms, 2);
    if (ctx->use_qjl) add(src->k_rnorms, dst->k_rnorms, 2);
    return r;
}

// ---- rows
// A block takes a run of 16-byte units of one stream and KV head, a thread one unit of all rows.  In place a row may be read
// by others after it was due to change, so a thread has loaded the unit of every row before it stores the first: up to
// kRegisterRows rows in registers, more in shared memory.
constexpr int kRegisterRows = 16;
constexpr int kMostShared = 224 * 1024;

struct RowArgs {
    Streams streams;
    int first_block[kStreams + 1];  // blocks of stream s: [first_block[s], first_block[s + 1])
    const int64_t *index;
    int rows, src_rows;
    int lo, hi;
    int64_t src_b, src_h, dst_b, dst_h;  // strides in tokens
    const int *seq_in;
    int *seq_out;
    bool in_place;
    int *error_flag;
};

// (Five blocks an SM: the registers that this leaves a thread keep more of its loads in flight; the case above 89.5 us without, 87.5 with, as single calls.)
template <bool STAGED> __global__ void __launch_bounds__(128, 5) tq_select_rows_kernel(const __grid_constant__ RowArgs a) {
    extern __shared__ uint4 stage[];  // [row][thread]
    const int h = blockIdx.y;
    int s = 0;
    while (s + 1 < a.streams.n && (int)blockIdx.x >= a.first_block[s + 1]) ++s;
    const Stream st = a.streams.s[s];
    const int64_t byte_lo = (int64_t)a.lo * st.token_bytes, byte_hi = (int64_t)a.hi * st.token_bytes;
    const int64_t unit = byte_lo / 16 + (int64_t)(blockIdx.x - a.first_block[s]) * blockDim.x + threadIdx.x;
    if (blockIdx.x == 0 && h == 0) {
        for (int b = threadIdx.x; b < a.rows; b += blockDim.x) {
            const int64_t from = a.index[b];
            const bool ok = from >= 0 && from < a.src_rows;
            if (!ok) atomicExch(a.error_flag, 7);
            if (a.seq_out) a.seq_out[b] = ok && a.seq_in ? a.seq_in[from] : ok || !a.in_place ? 0 : a.seq_in ? a.seq_in[b] : 0;
        }
    }
    if (unit * 16 >= byte_hi) return;
    const bool whole = unit * 16 >= byte_lo && unit * 16 + 16 <= byte_hi;  // (only norms have other units)
    const int64_t at = unit * 16 + h * a.src_h * st.token_bytes, to = unit * 16 + h * a.dst_h * st.token_bytes;
    // the source row of row b, or -1: nothing to do
    auto source = [&](int b) -> int64_t {
        const int64_t from = __ldg(a.index + b);
        return from < 0 || from >= a.src_rows || (a.in_place && from == b) ? -1 : from;
    };
    auto load = [&](int64_t from) { return *reinterpret_cast<const uint4 *>(st.src + at + from * a.src_b * st.token_bytes); };
    auto store = [&](int b, const uint4 &v) {
        uint8_t *p = st.dst + to + b * a.dst_b * st.token_bytes;
        if (whole) {
            *reinterpret_cast<uint4 *>(p) = v;
        } else {
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int64_t byte = unit * 16 + 2 * i;
                if (byte >= byte_lo && byte < byte_hi) reinterpret_cast<uint16_t *>(p)[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
            }
        }
    };
    if (STAGED) {
        for (int b = 0; b < a.rows; ++b) {
            const int64_t from = source(b);
            if (from >= 0) stage[b * blockDim.x + threadIdx.x] = load(from);
        }
        for (int b = 0; b < a.rows; ++b)
            if (source(b) >= 0) store(b, stage[b * blockDim.x + threadIdx.x]);
        return;
    }
    for (int b0 = 0; b0 < a.rows; b0 += kRegisterRows) {  // (one turn when in place)
        uint4 v[kRegisterRows];
        uint32_t live = 0;
#pragma unroll
        for (int i = 0; i < kRegisterRows; ++i) {
            const int64_t from = b0 + i < a.rows ? source(b0 + i) : -1;
            if (from >= 0) v[i] = load(from), live |= 1u << i;
        }
#pragma unroll
        for (int i = 0; i < kRegisterRows; ++i)
            if (live >> i & 1) store(b0 + i, v[i]);
    }
}

// ---- tokens
// A block per (batch entry, KV head); kGroupTokens tokens at a time pass through shared memory.  Paths ascend, so token i
// never lands behind its source, and what later groups read is not written before they have read it.
constexpr int kGroupTokens = 64;
constexpr int kKeepThreads = 256;

struct KeepArgs {
    Streams streams;
    const int *path, *counts, *lengths;
    int *lengths_out;
    int path_len, tree_start, capacity, kv_heads;
    int64_t stride_b, stride_h;
    int *error_flag;
};

__global__ void __launch_bounds__(kKeepThreads) tq_keep_tokens_kernel(const __grid_constant__ KeepArgs a) {
    __shared__ uint4 stage[kGroupTokens * 10];  // bytes of up to 64 tokens: at most 4 + 4 + 1 units and 6 bytes of norms each
    __shared__ int s_path[kGroupTokens];
    const int b = blockIdx.x / a.kv_heads, h = blockIdx.x % a.kv_heads;
    const int length = a.lengths[b], count = a.counts[b];
    const int *path = a.path + (int64_t)b * a.path_len;
    bool ok = length >= 0 && length <= a.tree_start && count >= 0 && count <= a.path_len;
    if (ok)
        for (int i = threadIdx.x; i < count; i += kKeepThreads)
            ok = ok && path[i] > (i ? path[i - 1] : -1) && path[i] < a.capacity - a.tree_start;
    ok = __syncthreads_and(ok);
    if (h == 0 && threadIdx.x == 0) {
        a.lengths_out[b] = ok ? length + count : length;
        if (!ok) atomicExch(a.error_flag, 7);
    }
    if (!ok) return;
    const int64_t row = b * a.stride_b + h * a.stride_h;
    for (int g = 0; g < count; g += kGroupTokens) {
        const int n = min(kGroupTokens, count - g);
        for (int i = threadIdx.x; i < n; i += kKeepThreads) s_path[i] = path[g + i];
        __syncthreads();
        for (int pass = 0; pass < 2; ++pass) {
            uint8_t *staged = reinterpret_cast<uint8_t *>(stage);
            for (int s = 0; s < a.streams.n; ++s) {
                const Stream &st = a.streams.s[s];
                const int64_t from = (row + a.tree_start) * st.token_bytes, to = (row + length + g) * st.token_bytes;
                if (st.token_bytes >= 16) {
                    const int units = st.token_bytes / 16;
                    for (int i = threadIdx.x; i < n * units; i += kKeepThreads) {
                        uint4 *mine = reinterpret_cast<uint4 *>(staged) + i;
                        if (pass == 0) *mine = *reinterpret_cast<const uint4 *>(st.src + from + (int64_t)s_path[i / units] * st.token_bytes + 16 * (i % units));
                        else *reinterpret_cast<uint4 *>(st.dst + to + 16 * i) = *mine;
                    }
                } else {
                    for (int i = threadIdx.x; i < n; i += kKeepThreads) {
                        uint16_t *mine = reinterpret_cast<uint16_t *>(staged) + i;
                        if (pass == 0) *mine = *reinterpret_cast<const uint16_t *>(st.src + from + 2 * (int64_t)s_path[i]);
                        else *reinterpret_cast<uint16_t *>(st.dst + to + 2 * i) = *mine;
                    }
                }
                staged += kGroupTokens * st.token_bytes;
            }
            __syncthreads();
        }
    }
}

}  // namespace

extern "C" int32_t tq_cache_select_rows(tq_ctx *ctx, const tq_cache_desc *src, const tq_cache_desc *dst, const int64_t *index,
                                        int32_t lo, int32_t hi, int32_t *seq_start_out, tq_stream stream) {
    TqRange range_("tq_cache_select_rows");
    if (!ctx || !index) return TQ_ERR_ARG;
    int rc = tq_check_cache(ctx, src);
    if (!rc) rc = tq_check_cache(ctx, dst);
    if (rc) return rc;
    if (src->kv_heads != dst->kv_heads || lo < 0 || hi < lo || hi > src->capacity || hi > dst->capacity) return TQ_ERR_ARG;
    if (((uintptr_t)index & 7) || ((uintptr_t)seq_start_out & 3)) return TQ_ERR_ARG;
    if (seq_start_out && (seq_start_out == src->seq_start || seq_start_out == dst->seq_start)) return TQ_ERR_ARG;
    RowArgs a = {};
    a.streams = streams_of(ctx, src, dst);
    int same = 0;
    for (int s = 0; s < a.streams.n; ++s) same += a.streams.s[s].src == a.streams.s[s].dst;
    if (same && (same != a.streams.n || src->batch != dst->batch || src->stride_b != dst->stride_b || src->stride_h != dst->stride_h))
        return TQ_ERR_ARG;  // a cache that shares some of its streams with the other, or sees them with other rows
    a.in_place = same != 0;
    a.index = index, a.rows = dst->batch, a.src_rows = src->batch, a.lo = lo, a.hi = hi;
    a.src_b = src->stride_b, a.src_h = src->stride_h, a.dst_b = dst->stride_b, a.dst_h = dst->stride_h;
    a.seq_in = src->seq_start, a.seq_out = seq_start_out;
    a.error_flag = ctx->error_flag;
    const bool staged = a.in_place && a.rows > kRegisterRows;
    int threads = 128;
    while (staged && threads > 32 && (int64_t)a.rows * threads * 16 > kMostShared) threads /= 2;
    if (staged && (int64_t)a.rows * threads * 16 > kMostShared) return TQ_ERR_UNSUPPORTED;
    const int smem = staged ? a.rows * threads * 16 : 0;
    int64_t blocks = 0;
    for (int s = 0; s < a.streams.n; ++s) {
        const int64_t bytes = a.streams.s[s].token_bytes;
        const int64_t units = (hi * bytes + 15) / 16 - lo * bytes / 16;
        a.first_block[s] = (int)blocks;
        blocks += (units + threads - 1) / threads;
    }
    if (blocks > 0x7fffffff || src->kv_heads > 65535) return TQ_ERR_UNSUPPORTED;
    a.first_block[a.streams.n] = (int)blocks;
    if (blocks == 0) blocks = 1;  // (no tokens: the row offsets alone)
    const dim3 grid((unsigned)blocks, (unsigned)src->kv_heads);
    if (staged) {
        TQ_CUDA_CHECK(tq_allow_shared<tq_select_rows_kernel<true>>(ctx->device, kMostShared));
        tq_select_rows_kernel<true><<<grid, threads, smem, (cudaStream_t)stream>>>(a);
    } else {
        tq_select_rows_kernel<false><<<grid, threads, 0, (cudaStream_t)stream>>>(a);
    }
    TQ_CUDA_CHECK(cudaGetLastError());
    return TQ_OK;
}

extern "C" int32_t tq_cache_keep_tokens(tq_ctx *ctx, const tq_cache_desc *cache, int32_t tree_start, const int32_t *path,
                                        int32_t path_len, const int32_t *counts, const int32_t *lengths, int32_t *lengths_out,
                                        tq_stream stream) {
    TqRange range_("tq_cache_keep_tokens");
    if (!ctx || !path || !counts || !lengths || !lengths_out) return TQ_ERR_ARG;
    const int rc = tq_check_cache(ctx, cache);
    if (rc) return rc;
    if (tree_start < 0 || tree_start > cache->capacity || path_len < 0 || lengths == lengths_out || counts == lengths_out) return TQ_ERR_ARG;
    if (((uintptr_t)path | (uintptr_t)counts | (uintptr_t)lengths | (uintptr_t)lengths_out) & 3) return TQ_ERR_ARG;
    if ((int64_t)cache->batch * cache->kv_heads > 0x7fffffff) return TQ_ERR_UNSUPPORTED;
    KeepArgs a = {};
    a.streams = streams_of(ctx, cache, cache);
    a.path = path, a.counts = counts, a.lengths = lengths, a.lengths_out = lengths_out;
    a.path_len = path_len, a.tree_start = tree_start, a.capacity = cache->capacity, a.kv_heads = cache->kv_heads;
    a.stride_b = cache->stride_b, a.stride_h = cache->stride_h, a.error_flag = ctx->error_flag;
    tq_keep_tokens_kernel<<<cache->batch * cache->kv_heads, kKeepThreads, 0, (cudaStream_t)stream>>>(a);
    TQ_CUDA_CHECK(cudaGetLastError());
    return TQ_OK;
}
