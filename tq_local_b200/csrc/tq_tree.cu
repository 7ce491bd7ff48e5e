// Attention of drafted tokens over the packed cache, on the 5th-generation tensor cores.  The T drafted tokens of every batch entry are
// packed at tokens [tree_start, tree_start + T); node i attends the entry's history [seq_start, length) and the drafted tokens that its
// mask names:
//
//   logit_ij = scale (kn_j c_k[codes_j] . (R_k q_i) + rn_j sqrt(pi/2)/D signs_j . (S q_i)),   out_i = R_v^T sum_j p_ij vn_j c_v[codes_j]
//
// Three launches.  The first rotates and projects the queries and rounds them to fp16 (the scale to base 2 and the sketch's factor folded in).
// The second attends: the 128 rows of a tile are (node, head of the group) pairs, its blocks of 128 are those of history and drafted tokens laid
// end to end, and all tiles' blocks laid end to end are cut into equal pieces, one a CTA (one CTA an SM).  The third joins a tile's pieces,
// un-rotates and rounds.  The second starts beside the first and turns packed tokens into operands before there are queries.
//
// Roles of the second.  Warps 0-7: softmax, half of a row's tokens a thread; the weights go back over the logits as 16-bit pairs.  Warps 8-23 turn packed
// tokens into fp16 operands in shared memory: centres times norm by a table of centre pairs, +-rn for the signs; half of them take the even blocks,
// half the odd ones.  Warp 24 issues the products, S = [Rq | Sq] [K | signs]^T with the queries in TMEM and O += P V.  Warp 25 requests the packed
// blocks (bulk copies, a ring of three).  TMEM: S of two blocks, O, the queries, 128 columns each.
//
// Roundings to fp16: the rotated queries, a centre, a centre times its norm, a weight; everything else is fp32.  Value centres are taken times the power of two
// that brings the largest to [1/2, 1): with the largest norm of fp16 they still fit, and norms down to 10^-4 stay clear of fp16's smallest numbers (a key
// operand's lost bits are lost to a logit in absolute terms, where they are nothing).  With fp16 outputs the error is
// 8e-4 relative to 64 bits (the output's own rounding 2e-4), with bf16 outputs 1.8e-3 (1.7e-3).  The largest share is that of the key operands: with the
// norms multiplied onto fp32 logits instead it is 5.5e-4, and 16 nodes over 8 x 32768 tokens take 221 us instead of 192.
//
// What bounds it: a block of 128 tokens takes a CTA 1.6 to 1.7 us whatever the bits, the sketch and the number of rows.  Of 195 us for 16 nodes over
// 8 x 32768 tokens (32 / 8 heads, 4 bits, sketch) leaving out the operands' stores gives back 48, the products 28, the look-ups 25, the exponentials 5; with
// all four left out 109 remain, which is the hand-over from role to role.  Shared memory is three quarters busy (operands written once and read once by the
// products, which read all of B again for every 128 rows).  Variants measured on the way: operands by eight warps straight from
// global memory, two stages of everything, 197 us; by sixteen, one block at a time, 247; two stages of values and two of the ring, 227.
// 896 threads are launched with 72 registers each, at which 184 to 232 bytes a thread are spilled.
#include <math.h>

#include <type_traits>

#include "tq_attn_tc.cuh"
#include "tq_step_blocks.cuh"

namespace {

constexpr int kRingSlots = 3;
constexpr int kSoftmaxWarps = 8, kOperandWarps = 16;  // and four more, of which one requests the packed blocks and one issues the products
constexpr int kThreads = 32 * (kSoftmaxWarps + kOperandWarps + 4);
constexpr int kBlock = 128;  // tokens of a block

struct TreeArgs {
    const uint8_t *k_codes, *k_signs, *v_codes;
    const uint16_t *k_norms, *k_rnorms, *v_norms;
    int64_t cache_sb, cache_sh;
    int capacity;  // tokens of a row (looked at by the bounds-checked build)
    int batch, kv_heads, group, nodes, tree_start;
    int positions, tiles, rows;  // nodes of a tile, tiles of a (batch entry, KV head), rows of a tile that hold something
    const int *seq_start, *lengths;
    const uint64_t *mask;
    const uint16_t *image_k, *image_s, *image_v;  // R_k, S, R_v
    float unscale_k, unscale_s, unscale_v;
    const float *centers_k, *centers_v;
    float cen_v_scale;  // power of two that brings the largest value centre to [1/2, 1), see the value operand
    const void *q;
    void *out;
    int64_t qb, qh, qt, ob, oh, ot;
    // Scratch, with a tile's rows innermost: lanes hold rows, and their 16 bytes lie side by side.
    uint4 *qop;       // [tile][16 or 32][rows] fp16, eight coordinates each
    float *part_ml;   // [piece][rows][2]
    float4 *part_o;   // [piece][32][rows]
    int ctas;
    int *error_flag;
};

// Where a coordinate lies in the operands and in O: the second and third eight of the last two quarters change places (see the stores below).
__device__ __forceinline__ int turned(int quarter, int eight) { return eight ^ (quarter & 2); }

// An entry's tokens as the kernel counts them: the cache's tokens from `first` (a multiple of eight, so that every stream can be copied in whole
// 16 bytes) up to the history's end, places up to the next multiple of eight, then the cache's tokens from tree_start, rounded down to one.
// The history is [lo, end), node 0 lies at nodes_at.
struct Entry {
    int first, lo, end, nodes_at;
};
__device__ __forceinline__ int up8(int n) { return (n + 7) & ~7; }
__device__ __forceinline__ Entry entry_of(const TreeArgs &a, int b) {
    const int length = a.lengths ? min(max(a.lengths[b], 0), a.tree_start) : a.tree_start;
    const int start = a.seq_start ? min(max(a.seq_start[b], 0), length) : 0;
    Entry e;
    e.first = start & ~7, e.lo = start - e.first, e.end = length - e.first, e.nodes_at = up8(e.end) + (a.tree_start & 7);
    return e;
}
// tokens that tile t of an entry may see, in blocks
__device__ __forceinline__ int tile_blocks(const TreeArgs &a, const Entry &e, int t) {
    const int drafted = a.mask ? a.nodes : min(a.nodes, (t + 1) * a.positions);
    return (e.nodes_at + drafted + kBlock - 1) / kBlock;
}
// How the blocks of all tiles, laid end to end, are cut into pieces of `chunk`, one a CTA.  Where there are no more tiles than CTAs a tile takes whole
// pieces (`whole`: its length is rounded up to them), if that costs at most two blocks a piece: going from one tile to the next takes a CTA some 5 us,
// as long as three blocks.
struct Cut {
    int64_t total;
    int chunk;
    bool whole;
    __device__ __forceinline__ int length(int blocks) const { return whole ? (blocks + chunk - 1) / chunk * chunk : blocks; }
};
__device__ __forceinline__ int64_t entry_length(const TreeArgs &a, const Cut &cut, int b) {  // of all heads' and tiles' blocks
    const Entry e = entry_of(a, b);
    int64_t n = 0;
    for (int t = 0; t < a.tiles; ++t) n += cut.length(tile_blocks(a, e, t));
    return n * a.kv_heads;
}
__device__ __forceinline__ Cut cut_of(const TreeArgs &a, int lane) {  // one warp
    auto sum = [&](const Cut &cut) {
        int64_t n = 0;
        for (int b = lane; b < a.batch; b += 32) n += entry_length(a, cut, b);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
        return n;
    };
    Cut cut = {0, 1, false};
    cut.total = sum(cut);
    cut.chunk = (int)((cut.total + a.ctas - 1) / a.ctas);
    if ((int64_t)a.batch * a.kv_heads * a.tiles <= a.ctas)
        for (int c = cut.chunk; c < cut.chunk + 3; ++c) {
            Cut trial = {0, c, true};
            trial.total = sum(trial);
            if (trial.total <= (int64_t)c * a.ctas) return trial;
        }
    return cut;
}

// ---------------------------------------------------------------------------------------------------- 128 x 128 matrices
// Rows times R_k^T, S^T or R_v, on the tensor core in two fp16 terms (see tq_umma.cuh).  A CTA takes up to 128 rows, so many that the
// CTAs fill the SMs once; four threads to a row, 32 coordinates each.
constexpr int kRowThreads = 512;

struct RowPlace {
    int b, h, head, node;  // head: of all query heads
    int64_t tile;
    int in;                // row of the tile
    bool live;
};
__device__ __forceinline__ RowPlace place_of(const TreeArgs &a, int64_t r, int64_t n_rows) {
    RowPlace p;
    p.in = (int)(r % a.rows), p.tile = r / a.rows;
    const int t = (int)(p.tile % a.tiles), g = p.in % a.group;
    p.h = (int)(p.tile / a.tiles % a.kv_heads), p.b = (int)(p.tile / a.tiles / a.kv_heads);
    p.head = p.h * a.group + g, p.node = t * a.positions + p.in / a.group;
    p.live = r < n_rows && p.node < a.nodes;
    return p;
}

// TMEM and the barriers of such a kernel, and its product: the rows are in TMEM as hi and lo terms at +256 and +320, the sums come at +0.
struct RowTile {
    uint32_t tmem, bar_image, bar_mma;
    bool lost = false;
    __device__ __forceinline__ void start(uint32_t *s_tmem, uint64_t *s_bars, uint32_t at, const uint16_t *image) {
        bar_image = smem_u32(s_bars), bar_mma = bar_image + 8;
        if (threadIdx.x < 32) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(s_tmem)), "r"(512));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n");
        }
        if (threadIdx.x == 32) {
            mbar_init(bar_image, 1), mbar_init(bar_mma, 1);
            asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            umma_load_image(at, image, bar_image);
        }
        umma_fence_before();
        __syncthreads();
        umma_fence_after();
        tmem = __shfl_sync(0xffffffffu, *s_tmem, 0);
    }
    // this thread's 32 coordinates of its row
    __device__ __forceinline__ void put(const float (&x)[32], int part, uint32_t lanes) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            uint32_t hi[8], lo[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) split_half2(f32x2(x[16 * c + 2 * i], x[16 * c + 2 * i + 1]), hi[i], lo[i]);
            tmem_st8(tmem + 256 + lanes + 16 * part + 8 * c, hi), tmem_st8(tmem + 320 + lanes + 16 * part + 8 * c, lo);
        }
        tmem_st_wait();
        umma_fence_before();
        __syncthreads();
    }
    template <bool TRANSPOSED> __device__ __forceinline__ void multiply(uint32_t image) {
        if (threadIdx.x < 32 && elect_one()) {
            umma_fence_after();
            if (!mbar_wait(bar_image, 0)) lost = true;
            umma_issue<2, TRANSPOSED>(tmem, tmem + 256, tmem + 320, image);
            umma_commit(bar_mma);
        }
        __syncwarp();
        if (!mbar_wait(bar_mma, 0)) lost = true;
        __syncwarp();
        umma_fence_after();
    }
    __device__ __forceinline__ void finish(int *error_flag) {
        if (lost) {  // the matrix may still be on its way, the product under way
            mbar_wait(bar_image, 0), mbar_wait(bar_mma, 0);
            atomicExch(error_flag, 8);
        }
        umma_fence_before();
        __syncthreads();
        if (threadIdx.x < 32) {
            umma_fence_after();
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512));
        }
    }
};

// Operand rows [Rq | Sq], blockIdx.y: which.  Sketch coordinates lie in the order in which the operand's signs do, (i, i + 16) of 32 side by side.
template <typename T, bool QJL> __global__ void __launch_bounds__(kRowThreads, 1) tq_tree_prep_kernel(const __grid_constant__ TreeArgs a, int64_t n_rows, int per_cta) {
    constexpr int kWide = QJL ? 256 : 128;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t s_bars[2];
    __shared__ uint32_t s_tmem;
    const uint32_t image = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const bool sketch = QJL && blockIdx.y;
    tq_launch_dependents();
    RowTile tile;
    tile.start(&s_tmem, s_bars, image, sketch ? a.image_s : a.image_k);
    const int row = threadIdx.x & 127, part = threadIdx.x >> 7;
    const uint32_t lanes = (uint32_t)(threadIdx.x & 96) << 16;
    const int64_t r = (int64_t)blockIdx.x * per_cta + row;
    const bool mine = row < per_cta && r < n_rows;
    float x[32] = {};
    if (mine) {
        const RowPlace p = place_of(a, r, n_rows);
        if (p.live) {
            const uint4 *src = reinterpret_cast<const uint4 *>(reinterpret_cast<const T *>(a.q) + p.b * a.qb + p.head * a.qh + p.node * a.qt) + 4 * part;
            const float scale = 0.08838834764831845f * 1.4426950408889634f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint4 v = __ldg(src + i);
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const T *pair = reinterpret_cast<const T *>(&w[e]);
                    x[8 * i + 2 * e] = tq_to_float<T>(pair[0]) * scale, x[8 * i + 2 * e + 1] = tq_to_float<T>(pair[1]) * scale;
                }
            }
        }
    }
    __syncwarp();
    tile.put(x, part, lanes);
    tile.multiply<false>(image);
    const float f = sketch ? a.unscale_s * (1.2533141373155003f / (float)TQ_D) : a.unscale_k;
    uint32_t y[32], o[16];
    tmem_ld32(tile.tmem + lanes + 32 * part, y);
    tmem_ld_wait(y);
#pragma unroll
    for (int e = 0; e < 16; ++e)
        o[e] = half2_bits(__uint_as_float(sketch ? y[e] : y[2 * e]) * f, __uint_as_float(sketch ? y[e + 16] : y[2 * e + 1]) * f);
    if (mine) {
        const int64_t to = r / a.rows * (kWide / 8) + (sketch ? 16 : 0) + 4 * part;
#pragma unroll
        for (int e = 0; e < 4; ++e) a.qop[(to + turned(part, e)) * a.rows + r % a.rows] = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
    }
    tile.finish(a.error_flag);
}

// ---------------------------------------------------------------------------------------------------- attention
// Shared memory: operands - two stages of keys, one of signs, one of values -, the tables of centre pairs, and a ring of packed blocks.  A slot of a
// table holds its pair once per lane, so that every lane reads its own bank.
template <int KB, int VB, bool QJL> struct Layout {
    static constexpr int kKeys = 0, kValues = 2 * kUmmaTermBytes, kSigns = 3 * kUmmaTermBytes;
    static constexpr int kKeyTable = kSigns + (QJL ? kUmmaTermBytes : 0), kValueTable = kKeyTable + 128 * (1 << 2 * KB);
    static constexpr int kRing = kValueTable + 128 * (1 << 2 * VB);
    // of a slot: the six streams
    static constexpr int kRawK = 0, kRawV = kRawK + kBlock * 16 * KB, kRawS = kRawV + kBlock * 16 * VB, kRawKN = kRawS + (QJL ? kBlock * 16 : 0),
                         kRawVN = kRawKN + 2 * kBlock, kRawRN = kRawVN + 2 * kBlock, kSlot = kRawRN + (QJL ? 2 * kBlock : 0);
    static constexpr int kTokenBytes = kSlot / kBlock;
    static constexpr int kBytes = kRing + kRingSlots * kSlot + 1024;
};

// Word i of the operand from 32 codes in BITS words (and one that is not looked at): two neighbouring codes by one look-up, times the norm.
template <int BITS> __device__ __forceinline__ uint32_t centre_pair(const uint32_t *words, int i, uint32_t lane_addr, uint32_t norm2) {
    constexpr uint32_t kMask = ((1u << 2 * BITS) - 1u) << 7;
    const int bit = 2 * BITS * i, w = bit >> 5, sh = bit & 31;
    uint32_t x;
    if (sh + 2 * BITS > 32) x = __funnelshift_r(words[w], words[w + 1], sh) << 7;
    else x = sh >= 7 ? words[w] >> (sh - 7) : words[w] << (7 - sh);
    uint32_t v;
    asm("ld.shared.u32 %0, [%1];\n" : "=r"(v) : "r"((x & kMask) + lane_addr));
    const __half2 r = __hmul2(*reinterpret_cast<const __half2 *>(&v), *reinterpret_cast<const __half2 *>(&norm2));
    return *reinterpret_cast<const uint32_t *>(&r);
}

// Bits [0, n) of a word, for any n.
__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }
// What a row sees of the 32 tokens from `at`: the history, then its nodes - mask, or as a chain the nodes [0, chain_end).
__device__ __forceinline__ uint32_t seen_word(const Entry &e, uint64_t mask, int chain_end, int at) {
    const uint32_t history = low_bits(e.end - at) & ~low_bits(e.lo - at);
    const int node = at - e.nodes_at;
    if (chain_end >= 0) return history | (low_bits(chain_end - node) & ~low_bits(-node));
    if (node <= -32 || node >= 64) return history;
    return history | (uint32_t)(node < 0 ? mask << -node : mask >> node);
}

template <int KB, int VB, bool QJL> __global__ void __launch_bounds__(kThreads, 1) tq_tree_kernel(const __grid_constant__ TreeArgs a) {
    using L = Layout<KB, VB, QJL>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t s_bars[2 + 2 + 2 + 2 + 1 + 1 + 1 + 2 + 2 * kRingSlots + 1];
    __shared__ uint32_t s_tmem;
    // What two warps that share rows tell each other, [block parity][half][row].  Two copies: one warp may be at the next block's logits while the other has
    // not yet read the maximum of this one (the products for them do not wait for this block's weights), but no further ahead than that.
    __shared__ float s_half[2][2][kUmmaRows];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t bars = smem_u32(s_bars);
    // kfull, vfull: operands are there; kfree, vfree: the products that read keys and signs, or values, are done; s: logits are there; p: weights are there; o: O += P V is
    // done; q: queries are there; raw, read: a slot of the ring is filled, has been read; done: see the end
    const uint32_t bar_kfull = bars, bar_kfree = bars + 16, bar_s = bars + 32, bar_p = bars + 48, bar_o = bars + 64, bar_q = bars + 72, bar_vfull = bars + 80, bar_vfree = bars + 88,
                   bar_raw = bars + 104, bar_read = bar_raw + 8 * kRingSlots, bar_done = bar_read + 8 * kRingSlots;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    constexpr int kProducts = kSoftmaxWarps + kOperandWarps;
    const int row_warps = (a.rows + 31) >> 5;  // quarters of the tile that have rows (the others' rows of S and O are what they are)
    if (warp == kProducts) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&s_tmem)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n");
    }
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar_kfull + 8 * i, kOperandWarps / 2), mbar_init(bar_kfree + 8 * i, 1), mbar_init(bar_vfree + 8 * i, 1);
            mbar_init(bar_s + 8 * i, 1), mbar_init(bar_p + 8 * i, 2 * row_warps);
        }
        mbar_init(bar_done, 1), mbar_init(bar_o, 1), mbar_init(bar_q, 2 * row_warps), mbar_init(bar_vfull, kOperandWarps / 2);
        for (int i = 0; i < kRingSlots; ++i) mbar_init(bar_raw + 8 * i, 1), mbar_init(bar_read + 8 * i, kOperandWarps / 2);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    {
        const float ck = a.centers_k[lane & 15], cv = a.centers_v[lane & 15] * a.cen_v_scale;
        auto fill = [&](uint32_t table, int bits, float centre) {
            for (int e = warp; e < 1 << 2 * bits; e += kThreads / 32) {
                const float lo = __shfl_sync(0xffffffffu, centre, e & ((1 << bits) - 1)), hi = __shfl_sync(0xffffffffu, centre, e >> bits);
                asm volatile("st.shared.u32 [%0], %1;\n" ::"r"(table + 128 * e + 4 * lane), "r"(half2_bits(lo, hi)) : "memory");
            }
        };
        fill(base + L::kKeyTable, KB, ck);
        fill(base + L::kValueTable, VB, cv);
    }
    // ---- this CTA's blocks: [flat, flat_end) of all tiles' blocks laid end to end.  (Counted here as well: packed tokens do not wait for the queries.)
    __shared__ Cut s_cut;
    __shared__ int64_t s_first;
    __shared__ int s_entry;
    if (warp == 0) {
        const Cut cut = cut_of(a, lane);
        const int64_t from = (int64_t)blockIdx.x * cut.chunk;
        int64_t before = 0;
        for (int b0 = 0; from < cut.total && b0 < a.batch; b0 += 32) {  // the entry that holds block `from`
            const int64_t mine = b0 + lane < a.batch ? entry_length(a, cut, b0 + lane) : 0;
            int64_t end = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t x = __shfl_up_sync(0xffffffffu, end, o);
                if (lane >= o) end += x;
            }
            const bool here = before + end - mine <= from && from < before + end;
            if (here) s_entry = b0 + lane, s_first = before + end - mine;
            before += __shfl_sync(0xffffffffu, end, 31);
            if (__any_sync(0xffffffffu, here)) break;
        }
        if (lane == 0) s_cut = cut;
    }
    umma_fence_before();
    __syncthreads();
    umma_fence_after();
    tq_launch_dependents();
    const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0), t_o = tmem + 256, t_q = tmem + 384;
    const Cut cut = s_cut;
    int64_t flat = (int64_t)blockIdx.x * cut.chunk;
    const int64_t flat_end = min(flat + cut.chunk, cut.total);
    int b_at = 0;
    int64_t b_first = 0, b_next = 0;
    if (flat < flat_end) b_at = s_entry, b_first = s_first, b_next = b_first + entry_length(a, cut, b_at);
    struct Segment {  // the part of one tile inside this CTA's piece: blocks [k, k_end)
        int b, h, t, k, k_end;
        Entry e;
        int64_t tile;
    };
    auto next_segment = [&]() {
        while (flat >= b_next) ++b_at, b_first = b_next, b_next += entry_length(a, cut, b_at);
        Segment g;
        g.e = entry_of(a, b_at), g.b = b_at;
        const int per_head = (int)((b_next - b_first) / a.kv_heads);
        int in = (int)(flat - b_first);
        g.h = in / per_head, in -= g.h * per_head;
        int nb = tile_blocks(a, g.e, 0);
        for (g.t = 0; in >= cut.length(nb);) in -= cut.length(nb), ++g.t, nb = tile_blocks(a, g.e, g.t);
        const int64_t left = flat_end - flat;
        const int end = left < cut.length(nb) - in ? in + (int)left : cut.length(nb);
        flat += end - in;
        g.k = in, g.k_end = min(end, nb);
        g.tile = ((int64_t)g.b * a.kv_heads + g.h) * a.tiles + g.t;
        return g;
    };
    bool lost = false;  // a wait of this thread ran out: it waits for nothing more
    auto wait = [&](uint32_t bar, uint32_t parity) {
        if (!lost && !mbar_wait(bar, parity)) lost = true;
    };
    uint32_t asked = 0;  // packed blocks that were requested

    if (warp >= kProducts) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;\n");
        if (warp == kProducts) {
            // ---------------- products, by one thread; n counts blocks since the kernel began
            if (elect_one()) {
                constexpr uint32_t instr_s = umma_instr<false>(), instr_o = umma_instr<true>();
                auto scores = [&](uint32_t n) {
                    wait(bar_kfull + 8 * (n & 1), n >> 1 & 1);
                    umma_fence_after();
#pragma unroll
                    for (int part = 0; part < (QJL ? 2 : 1); ++part) {
                        const uint64_t desc = umma_desc<false>(base + (part ? L::kSigns : L::kKeys + (n & 1) * kUmmaTermBytes));
#pragma unroll
                        for (uint32_t s = 0; s < 8; ++s)
                            umma_f16(tmem + 128 * (n & 1), t_q + 64 * part + 8 * s, desc + (((s >> 2) * kUmmaSlabBytes + (s & 3) * 32) >> 4), instr_s, part | (s > 0));
                    }
                    umma_commit(bar_s + 8 * (n & 1));
                    umma_commit(bar_kfree + 8 * (n & 1));
                };
                uint32_t n = 0, segment = 0;
                while (flat < flat_end) {
                    const Segment g = next_segment();
                    const uint32_t end = n + (g.k_end - g.k);
                    wait(bar_q, segment++ & 1);
                    scores(n);
                    for (bool first = true; n < end; ++n, first = false) {
                        if (n + 1 < end) scores(n + 1);
                        wait(bar_vfull, n & 1);
                        wait(bar_p + 8 * (n & 1), n >> 1 & 1);
                        umma_fence_after();
                        attn_values(t_o, tmem + 128 * (n & 1), base + L::kValues, instr_o, !first);
                        umma_commit(bar_vfree + 8 * (n & 1));
                        umma_commit(bar_o);
                    }
                }
            }
        } else if (warp == kProducts + 1) {
            // ---------------- packed blocks: bulk copies of whole eights of tokens, kRingSlots blocks ahead
            if (elect_one()) {
                uint32_t &n = asked;
                while (flat < flat_end && !lost) {
                    const Segment g = next_segment();
                    const int64_t row = g.b * a.cache_sb + g.h * a.cache_sh;
                    const int tree = up8(g.e.end), tree_end = tree + up8((a.tree_start & 7) + a.nodes);  // places of the second run of tokens
                    for (int k = g.k; k < g.k_end; ++k, ++n) {
                        const int slot = n % kRingSlots, at = k * kBlock;
                        if (n >= kRingSlots) wait(bar_read + 8 * slot, (n / kRingSlots & 1) ^ 1);
                        if (lost) break;
                        const uint32_t bar = bar_raw + 8 * slot, dst = base + L::kRing + slot * L::kSlot;
                        const int n0 = max(min(kBlock, tree - at), 0), n1 = max(min(kBlock, tree_end - at) - n0, 0);
#ifdef TQ_DEBUG_BOUNDS
                        // Both runs of tokens lie inside their row and the slot inside shared memory; what does not is recorded (status 6) and left out.
                        uint32_t dyn_size;
                        asm("mov.u32 %0, %%dynamic_smem_size;\n" : "=r"(dyn_size));
                        const int t0 = g.e.first + at, t1 = (a.tree_start & ~7) + at + n0 - tree;
                        if (g.b < 0 || g.b >= a.batch || g.h < 0 || g.h >= a.kv_heads || n0 + n1 <= 0 || n0 + n1 > kBlock || ((n0 | n1) & 7) ||
                            (n0 && (t0 < 0 || t0 + n0 > a.capacity)) || (n1 && (t1 < 0 || t1 + n1 > a.capacity)) ||
                            dst + L::kSlot > smem_u32(smem_raw) + dyn_size) {
                            atomicExch(a.error_flag, 6);
                            mbar_arrive_one(bar);
                            continue;
                        }
#endif
                        mbar_expect_tx(bar, (n0 + n1) * L::kTokenBytes);
                        auto run = [&](int to, int64_t t, int count) {
                            tma_load_1d(dst + L::kRawK + to * 16 * KB, a.k_codes + t * 16 * KB, count * 16 * KB, bar);
                            tma_load_1d(dst + L::kRawV + to * 16 * VB, a.v_codes + t * 16 * VB, count * 16 * VB, bar);
                            tma_load_1d(dst + L::kRawKN + to * 2, a.k_norms + t, count * 2, bar);
                            tma_load_1d(dst + L::kRawVN + to * 2, a.v_norms + t, count * 2, bar);
                            if (QJL) {
                                tma_load_1d(dst + L::kRawS + to * 16, a.k_signs + t * 16, count * 16, bar);
                                tma_load_1d(dst + L::kRawRN + to * 2, a.k_rnorms + t, count * 2, bar);
                            }
                        };
                        if (n0) run(0, row + g.e.first + at, n0);
                        if (n1) run(n0, row + (a.tree_start & ~7) + at + n0 - tree, n1);
                    }
                }
            }
        }
    } else if (warp >= kSoftmaxWarps) {
        // ---------------- operands.  Half of the warps take the even blocks, half the odd ones, so that one half's waits pass behind the other's
        // work.  A quarter of two tokens' coordinates a thread, four lanes to a token.
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;\n");
        const uint32_t half = (uint32_t)(warp - kSoftmaxWarps) / (kOperandWarps / 2);
        const int quarter = lane & 3, row0 = 16 * ((warp - kSoftmaxWarps) % (kOperandWarps / 2)) + (lane >> 2);  // and row0 + 8
        const uint32_t lane_k = base + L::kKeyTable + 4 * lane, lane_v = base + L::kValueTable + 4 * lane;
        // Eight lanes store two tokens' quarters: with the last two quarters' eights turned, to eight different banks of 16 bytes.
        const uint32_t turn = (quarter & 1) * 4 ^ (quarter & 2) ^ (row0 & 7);
        const uint32_t my_row = base + (quarter >> 1) * kUmmaSlabBytes + (row0 >> 3) * 1024 + (row0 & 7) * 128;
        auto put = [&](uint32_t at, auto word) {
#pragma unroll
            for (int c = 0; c < 4; ++c) sts128(my_row + at + ((c ^ turn) << 4), word(4 * c), word(4 * c + 1), word(4 * c + 2), word(4 * c + 3));
        };
        auto words = [&](uint32_t src, auto count, uint32_t *w) {
            constexpr int n = decltype(count)::value;
            if constexpr (n == 4) {
                const uint4 x = lds128(src);
                w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
            } else {
#pragma unroll
                for (int i = 0; i < n; ++i) asm volatile("ld.shared.u32 %0, [%1];\n" : "=r"(w[i]) : "r"(src + 4 * i) : "memory");
            }
            w[n] = 0;
        };
        auto norm2 = [&](uint32_t src, bool token) {  // (what is no token holds anything)
            uint16_t x;
            asm volatile("ld.shared.u16 %0, [%1];\n" : "=h"(x) : "r"(src) : "memory");
            return token ? x * 0x10001u : 0u;
        };
        uint32_t n = 0;
        while (flat < flat_end) {
            const Segment g = next_segment();
            for (int k = g.k; k < g.k_end; ++k, ++n) {
                if ((n & 1) != half) continue;
                const int slot = n % kRingSlots;
                const uint32_t raw = base + L::kRing + slot * L::kSlot, stage = L::kKeys + half * kUmmaTermBytes;
                auto token = [&](int i) {
                    const int v = k * kBlock + row0 + 8 * i;
                    return (v >= g.e.lo && v < g.e.end) || (v >= g.e.nodes_at && v < g.e.nodes_at + a.nodes);
                };
                wait(bar_raw + 8 * slot, n / kRingSlots & 1);
                if (n > 1) wait(bar_kfree + 8 * half, (n >> 1 & 1) ^ 1);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int row = row0 + 8 * i;
                    uint32_t w[KB + 1];
                    words(raw + L::kRawK + row * 16 * KB + 4 * KB * quarter, std::integral_constant<int, KB>(), w);
                    const uint32_t norm = norm2(raw + L::kRawKN + 2 * row, token(i));
                    put(stage + 1024 * i, [&](int j) { return centre_pair<KB>(w, j, lane_k, norm); });
                }
                if (QJL) {
                    if (n) wait(bar_kfree + 8 * (half ^ 1), (n - 1) >> 1 & 1);  // (the signs have one stage)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int row = row0 + 8 * i;
                        uint32_t w[2];
                        words(raw + L::kRawS + row * 16 + 4 * quarter, std::integral_constant<int, 1>(), w);
                        const uint32_t norm = norm2(raw + L::kRawRN + 2 * row, token(i)) ^ 0x80008000u;
                        put(L::kSigns + 1024 * i, [&](int j) { return ((w[0] << (15 - j)) & 0x80008000u) ^ norm; });  // signs j and j + 16; a set bit is +
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                mbar_arrive_warp(bar_kfull + 8 * half);
                uint32_t vw[2][VB + 1], vn2[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int row = row0 + 8 * i;
                    words(raw + L::kRawV + row * 16 * VB + 4 * VB * quarter, std::integral_constant<int, VB>(), vw[i]);
                    vn2[i] = norm2(raw + L::kRawVN + 2 * row, token(i));
                }
                mbar_arrive_warp(bar_read + 8 * slot);
                if (n) wait(bar_vfree + 8 * (half ^ 1), (n - 1) >> 1 & 1);  // (the values have one stage)
#pragma unroll
                for (int i = 0; i < 2; ++i) put(L::kValues + 1024 * i, [&](int j) { return centre_pair<VB>(vw[i], j, lane_v, vn2[i]); });
                asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                mbar_arrive_warp(bar_vfull);
            }
        }
    } else {
        // ---------------- softmax: half of a row's tokens, and of its output's coordinates, a thread
        asm volatile("setmaxnreg.inc.sync.aligned.u32 104;\n");
        const int half = warp >> 2, row = tid & 127;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, t_mine = t_o + lanes + 64 * half;
        constexpr int kWide = QJL ? 256 : 128;
        // the two warps that share 32 rows
        auto pair_sync = [&]() { asm volatile("bar.sync %0, 64;\n" ::"r"(1 + (warp & 3)) : "memory"); };
        auto load_queries = [&](int64_t t) {  // of tile t
            const uint4 *src = a.qop + (t * (kWide / 8) + kWide / 16 * half) * a.rows + row;
            uint32_t q[kWide / 4];
#pragma unroll
            for (int e = 0; e < kWide / 16; ++e) {
                const uint4 x = row < a.rows ? src[e * a.rows] : make_uint4(0, 0, 0, 0);
                q[4 * e] = x.x, q[4 * e + 1] = x.y, q[4 * e + 2] = x.z, q[4 * e + 3] = x.w;
            }
            __syncwarp();
#pragma unroll
            for (int i = 0; i < kWide / 128; ++i) tmem_st32(t_q + lanes + kWide / 4 * half + 32 * i, q + 32 * i);
            tmem_st_wait();
            umma_fence_before();
            mbar_arrive_warp(bar_q);
        };
        uint32_t n = 0;
        tq_grid_dependency_wait();  // (the queries)
        const bool any = (warp & 3) < row_warps && flat < flat_end;
        Segment next = {};
        if (any) next = next_segment(), load_queries(next.tile);
        if (any) for (bool more = true; more;) {
            const Segment g = next;
            const int node = g.t * a.positions + row / a.group;
            const bool live = row < a.rows && node < a.nodes;
            const uint64_t mask = live && a.mask ? a.mask[(int64_t)g.b * a.nodes + node] & (~0ull >> (64 - a.nodes)) : 0;
            const int chain_end = a.mask ? -1 : live ? node + 1 : 0;
            float m_ref = -INFINITY;
            uint64_t sum[2] = {0, 0};
            for (int k = g.k; k < g.k_end; ++k, ++n) {
                const uint32_t t_s = tmem + 128 * (n & 1) + lanes;
                wait(bar_s + 8 * (n & 1), n >> 1 & 1);
                __syncwarp();
                umma_fence_after();
                uint32_t s[64];
                tmem_ld32(t_s + 64 * half, s), tmem_ld32(t_s + 64 * half + 32, s + 32);
                tmem_ld_wait(s), tmem_ld_wait(s + 32);
                if ((k + 1) * kBlock > g.e.end || k * kBlock < g.e.lo) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const uint32_t seen = seen_word(g.e, mask, chain_end, k * kBlock + 64 * half + 32 * x);
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (!(seen >> i & 1)) s[32 * x + i] = 0xff800000u;
                    }
                }
                float top[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) top[i] = max3(__uint_as_float(s[i]), __uint_as_float(s[i + 4]), __uint_as_float(s[i + 8]));
#pragma unroll
                for (int i = 12; i < 60; i += 8)
#pragma unroll
                    for (int e = 0; e < 4; ++e) top[e] = max3(top[e], __uint_as_float(s[i + e]), __uint_as_float(s[i + e + 4]));
                const float last = max3(__uint_as_float(s[60]), __uint_as_float(s[61]), fmaxf(__uint_as_float(s[62]), __uint_as_float(s[63])));
                float peak = max3(max3(top[0], top[1], top[2]), top[3], last);
                s_half[n & 1][half][row] = peak;
                umma_fence_before();
                pair_sync();  // (both have read their logits as well: the weights go over them)
                umma_fence_after();
                peak = fmaxf(peak, s_half[n & 1][half ^ 1][row]);
                if (k == g.k) {
                    m_ref = peak;
                } else {
                    const bool raise = live && peak - m_ref > kLag;
                    if (__any_sync(0xffffffffu, raise)) {
                        float keep = 1.f;
                        if (raise) keep = exp2_hw(m_ref - peak), m_ref = peak;
                        const uint64_t keep2 = f32x2(keep, keep);
                        sum[0] = f32x2_mul(sum[0], keep2), sum[1] = f32x2_mul(sum[1], keep2);
                        wait(bar_o, (n - 1) & 1);  // the values of the block before
                        __syncwarp();
                        umma_fence_after();
#pragma unroll 1
                        for (int i = 0; i < 4; ++i) {
                            uint32_t o[16];
                            tmem_ld16(t_mine + 16 * i, o);
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                            tmem_st16(t_mine + 16 * i, o);
                        }
                    }
                }
                const float shift = m_ref == -INFINITY ? 0.f : -m_ref;
                const uint64_t shift2 = f32x2(shift, shift);
#pragma unroll
                for (int part = 0; part < 2; ++part) {
                    uint32_t p[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float x, y;
                        f32x2_split(f32x2_add(f32x2(__uint_as_float(s[32 * part + 2 * i]), __uint_as_float(s[32 * part + 2 * i + 1])), shift2), x, y);
                        x = exp2_hw(x), y = exp2_hw(y);
                        sum[i & 1] = f32x2_add(sum[i & 1], f32x2(x, y));
                        p[i] = pack16<false>(x, y);
                    }
                    tmem_st16(t_s + 32 * half + 16 * part, p);
                }
                tmem_st_wait();
                umma_fence_before();
                // (the wait for the last values tells them from those before only if these are known to be done)
                if (k > g.k && k + 1 == g.k_end) wait(bar_o, (n - 1) & 1);
                mbar_arrive_warp(bar_p + 8 * (n & 1));
            }
            // ---- the next queries, so that their first products run beside what follows (those that read the ones before are done: their logits were here)
            more = flat < flat_end;
            if (more) next = next_segment(), load_queries(next.tile);
            // ---- this piece of the tile's rows
            float l0, l1;
            f32x2_split(f32x2_add(sum[0], sum[1]), l0, l1);
            pair_sync();  // (the last peak has been read)
            s_half[0][half][row] = l0 + l1;
            pair_sync();
            const float l = s_half[0][0][row] + s_half[0][1][row];
            wait(bar_o, (n - 1) & 1);
            __syncwarp();
            umma_fence_after();
            const int64_t r = (g.tile + blockIdx.x) * a.rows + row;
#ifdef TQ_DEBUG_BOUNDS
            const bool known = r >= 0 && r < ((int64_t)a.batch * a.kv_heads * a.tiles + a.ctas) * a.rows;  // a piece that the workspace has
            if (live && !known) atomicExch(a.error_flag, 6);
#else
            constexpr bool known = true;
#endif
            if (known && live && half == 0) *reinterpret_cast<float2 *>(a.part_ml + 2 * r) = make_float2(m_ref, l);
#pragma unroll 1
            for (int i = 0; i < 2; ++i) {
                uint32_t o[32];
                __syncwarp();
                tmem_ld32(t_mine + 32 * i, o);
                tmem_ld_wait(o);
                if (known && live)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        a.part_o[((g.tile + blockIdx.x) * 32 + 16 * half + 8 * i + e) * a.rows + row] =
                            make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]), __uint_as_float(o[4 * e + 2]), __uint_as_float(o[4 * e + 3]));
            }
            umma_fence_before();
            pair_sync();  // (the sums have been read)
        }
    }
    umma_fence_before();
    if (__syncthreads_or(lost)) {
        // A thread whose wait ran out waits for nothing more.  What was set going ends before the CTA does all the same: a copy that landed later would land in
        // another's shared memory.
        if (lost) atomicExch(a.error_flag, 8);
        if (warp == kProducts && elect_one()) {
            umma_commit(bar_done);
            mbar_wait(bar_done, 0);
        } else if (warp == kProducts + 1 && elect_one()) {
            for (uint32_t i = asked > kRingSlots ? asked - kRingSlots : 0; i < asked; ++i) mbar_wait(bar_raw + 8 * (i % kRingSlots), i / kRingSlots & 1);
        }
        __syncthreads();
    }
    if (warp == kProducts) {
        umma_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512));
    }
}

// ---------------------------------------------------------------------------------------------------- join
// Merges a row's pieces, brings its largest coordinate to [2^13, 2^14) for the fp16 terms, un-rotates and rounds.
// Where a CTA has few rows, the pieces of a row are shared out: thread (slot, part) takes every `groups`-th piece of row slot % rows.
template <typename T> __global__ void __launch_bounds__(kRowThreads, 1) tq_tree_join_kernel(const __grid_constant__ TreeArgs a, int64_t n_rows, int per_cta) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t s_bars[2];
    __shared__ uint32_t s_tmem;
    __shared__ float s_most[4][128];
    __shared__ float2 s_ml[128];
    __shared__ Cut s_cut;
    __shared__ float s_sum[128];
    const uint32_t image = (smem_u32(smem_raw) + 1023u) & ~1023u;
    float4 *const s_part = reinterpret_cast<float4 *>(smem_raw + (image - smem_u32(smem_raw)) + kUmmaImageBytes);  // [slot][33]
    RowTile tile;
    tile.start(&s_tmem, s_bars, image, a.image_v);
    const int slot = threadIdx.x & 127, part = threadIdx.x >> 7;
    const uint32_t lanes = (uint32_t)(threadIdx.x & 96) << 16;
    int rows = 8;
    while (rows < per_cta) rows *= 2;
    const int groups = kUmmaRows / rows, row = slot & (rows - 1), group = slot / rows;
    const int64_t r = (int64_t)blockIdx.x * per_cta + row;
    RowPlace p = {};
    if (row < per_cta && r < n_rows) p = place_of(a, r, n_rows);
    // which pieces a row has: counted again, while the second launch runs
    if (threadIdx.x < 32) {
        const Cut cut = cut_of(a, threadIdx.x);
        if (threadIdx.x == 0) s_cut = cut;
    }
    __syncthreads();
    int64_t piece0 = 0;
    int n = 0;
    if (p.live) {
        const Cut cut = s_cut;
        const Entry e = entry_of(a, p.b);
        const int t = (int)(p.tile % a.tiles), nb = tile_blocks(a, e, t);
        int64_t first = entry_length(a, cut, p.b) / a.kv_heads * p.h;
        for (int b = 0; b < p.b; ++b) first += entry_length(a, cut, b);
        for (int x = 0; x < t; ++x) first += cut.length(tile_blocks(a, e, x));
        const int64_t c0 = first / cut.chunk;
        piece0 = p.tile + c0, n = (int)((first + nb - 1) / cut.chunk - c0) + 1;
    }
    tq_grid_dependency_wait();
    float o[32] = {};
    float m = -INFINITY, l = 0.f;
    if (p.live) {
#pragma unroll 2
        for (int c = group; c < n; c += groups) {
            const float2 x = reinterpret_cast<const float2 *>(a.part_ml)[(piece0 + c) * a.rows + p.in];
            const float4 *src = a.part_o + ((piece0 + c) * 32 + 8 * part) * a.rows + p.in;
            float4 v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = src[(2 * turned(part, i >> 1) + (i & 1)) * a.rows];
            if (x.y == 0.f) continue;  // (a piece in which the row saw nothing)
            const float top = fmaxf(m, x.x), keep = exp2f(m - top), f = exp2f(x.x - top);
            m = top, l = l * keep + f * x.y;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                o[4 * i] = o[4 * i] * keep + f * v[i].x, o[4 * i + 1] = o[4 * i + 1] * keep + f * v[i].y;
                o[4 * i + 2] = o[4 * i + 2] * keep + f * v[i].z, o[4 * i + 3] = o[4 * i + 3] * keep + f * v[i].w;
            }
        }
    }
    if (groups > 1) {
        if (part == 0) s_ml[slot] = make_float2(m, l);
#pragma unroll
        for (int i = 0; i < 8; ++i) s_part[slot * 33 + 8 * part + i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        __syncthreads();
        for (int i = threadIdx.x; i < rows * 32; i += kRowThreads) {  // four coordinates of a row, from its groups
            const int r0 = i >> 5, c = i & 31;
            float top = -INFINITY, sum = 0.f;
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int x = 0; x < groups; ++x) top = fmaxf(top, s_ml[x * rows + r0].x);
            for (int x = 0; x < groups; ++x) {
                const float2 ml = s_ml[x * rows + r0];
                const float f = ml.y == 0.f ? 0.f : exp2f(ml.x - top);
                const float4 v = s_part[(x * rows + r0) * 33 + c];
                sum += f * ml.y;
                y = make_float4(y.x + f * v.x, y.y + f * v.y, y.z + f * v.z, y.w + f * v.w);
            }
            s_part[r0 * 33 + c] = y;  // (nobody else reads these of group 0)
            if (c == 0) s_sum[r0] = sum;
        }
        __syncthreads();
        l = group == 0 ? s_sum[row] : 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float4 v = group == 0 ? s_part[row * 33 + 8 * part + i] : make_float4(0.f, 0.f, 0.f, 0.f);
            o[4 * i] = v.x, o[4 * i + 1] = v.y, o[4 * i + 2] = v.z, o[4 * i + 3] = v.w;
        }
        p.live = p.live && group == 0;
    }
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) o[i] *= inv;
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) most = fmaxf(most, fabsf(o[i]));
    s_most[part][slot] = most;
    __syncthreads();
    most = fmaxf(fmaxf(s_most[0][slot], s_most[1][slot]), fmaxf(s_most[2][slot], s_most[3][slot]));
    // the power of two from the exponent's bits; what is too small for one is left as it is, and so is infinity
    const int exponent = (int)(__float_as_uint(most) >> 23);
    const int up = exponent == 0 || exponent == 255 ? 0 : min(13 + 127 - exponent, 120);
    const float raise = __uint_as_float((uint32_t)(127 + up) << 23), lower = __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
    for (int i = 0; i < 32; ++i) o[i] *= raise;
    __syncwarp();
    tile.put(o, part, lanes);
    tile.multiply<true>(image);
    uint32_t y[32];
    tmem_ld32(tile.tmem + lanes + 32 * part, y);
    tmem_ld_wait(y);
    if (p.live) {
        const float f = a.unscale_v * lower;
        uint4 *dst = reinterpret_cast<uint4 *>(reinterpret_cast<T *>(a.out) + p.b * a.ob + p.head * a.oh + p.node * a.ot + 32 * part);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                w[e] = pack16<std::is_same<T, __nv_bfloat16>::value>(__uint_as_float(y[8 * i + 2 * e]) * f, __uint_as_float(y[8 * i + 2 * e + 1]) * f);
            dst[i] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    tile.finish(a.error_flag);
}

bool aligned(const tq_dense_desc *d) {
    return !(((uintptr_t)d->data | (uintptr_t)(2 * (d->stride_b | d->stride_h | d->stride_t))) & 15);
}

struct Plan {
    int positions, tiles, rows, ctas;
    int64_t n_tiles;
    size_t qop, ml, o, bytes;  // workspace offsets
};
Plan plan(const tq_ctx *ctx, int64_t batch, int q_heads, int kv_heads, int nodes, int tree_start) {
    Plan p;
    const int group = q_heads / kv_heads;
    p.positions = kUmmaRows / group;
    p.tiles = (nodes + p.positions - 1) / p.positions;
    p.rows = (nodes < p.positions ? nodes : p.positions) * group;
    p.n_tiles = batch * kv_heads * p.tiles;
    const int64_t most = p.n_tiles * (((int64_t)tree_start + nodes + 21 + kBlock - 1) / kBlock);  // (with the places between, see Entry)
    // A CTA an SM.  (Those of the first launch's few CTAs left out, so that none of the second waits for one: 12 nodes behind 65536 tokens, 32 / 8
    // heads, 77.3 us instead of 74.3, 4 x 4099 tokens and one node 33.6 instead of 33.3, 8191 and 12 29.9 instead of 30.0.)
    p.ctas = most < ctx->sm_count ? (int)most : ctx->sm_count;
    auto take = [at = (size_t)0](size_t bytes) mutable {
        const size_t r = at;
        at += (bytes + 255) / 256 * 256;
        return r;
    };
    const size_t pieces = (size_t)(p.n_tiles + p.ctas) * p.rows;
    p.qop = take((size_t)p.n_tiles * p.rows * (ctx->use_qjl ? 512 : 256));
    p.ml = take(pieces * 2 * sizeof(float));
    p.o = take(pieces * TQ_D * sizeof(float));
    p.bytes = take(0);
    return p;
}

template <int KB, int VB, bool QJL> cudaError_t launch_attend(const TreeArgs &a, int device, cudaStream_t stream) {
    constexpr int smem = Layout<KB, VB, QJL>::kBytes;
    const cudaError_t e = tq_allow_shared<tq_tree_kernel<KB, VB, QJL>>(device, smem);
    return e != cudaSuccess ? e : tq_launch_kernel(tq_tree_kernel<KB, VB, QJL>, dim3(a.ctas), dim3(kThreads), smem, stream, true, a);
}

template <typename T, bool QJL> cudaError_t launch_prep(const TreeArgs &a, int64_t n_rows, unsigned blocks, int per_cta, int device, cudaStream_t stream) {
    constexpr int smem = kUmmaImageBytes + 1024;
    const cudaError_t e = tq_allow_shared<tq_tree_prep_kernel<T, QJL>>(device, smem);
    return e != cudaSuccess ? e : tq_launch_kernel(tq_tree_prep_kernel<T, QJL>, dim3(blocks, QJL ? 2 : 1), dim3(kRowThreads), smem, stream, false, a, n_rows, per_cta);
}

template <typename T> cudaError_t launch(const TreeArgs &a, const tq_ctx *ctx, int64_t n_rows, cudaStream_t stream) {
    const bool qjl = ctx->use_qjl != 0;
    const int device = ctx->device;
    const int64_t share = ((n_rows + ctx->sm_count - 1) / ctx->sm_count + 7) / 8 * 8;
    const int per_cta = share < kUmmaRows ? (int)share : kUmmaRows;
    const unsigned blocks = (unsigned)((n_rows + per_cta - 1) / per_cta);
    const unsigned prep_blocks = (unsigned)((n_rows + kUmmaRows - 1) / kUmmaRows);  // (few CTAs: the others of the second launch do not wait for their SMs)
    cudaError_t e = qjl ? launch_prep<T, true>(a, n_rows, prep_blocks, kUmmaRows, device, stream) : launch_prep<T, false>(a, n_rows, prep_blocks, kUmmaRows, device, stream);
    if (e != cudaSuccess) return e;
    switch (ctx->bits) {
        case 2: e = qjl ? launch_attend<1, 2, true>(a, device, stream) : launch_attend<2, 2, false>(a, device, stream); break;
        case 3: e = qjl ? launch_attend<2, 3, true>(a, device, stream) : launch_attend<3, 3, false>(a, device, stream); break;
        case 4: e = qjl ? launch_attend<3, 4, true>(a, device, stream) : launch_attend<4, 4, false>(a, device, stream); break;
        default: return cudaErrorInvalidValue;
    }
    if (e != cudaSuccess) return e;
    constexpr int smem = kUmmaImageBytes + kUmmaRows * 33 * 16 + 1024;
    e = tq_allow_shared<tq_tree_join_kernel<T>>(device, smem);
    return e != cudaSuccess ? e : tq_launch_kernel(tq_tree_join_kernel<T>, dim3(blocks), dim3(kRowThreads), smem, stream, true, a, n_rows, per_cta);
}

}  // namespace

extern "C" size_t tq_tree_workspace_bytes(tq_ctx *ctx, int32_t batch, int32_t q_heads, int32_t kv_heads, int32_t n_nodes, int32_t tree_start) {
    if (!ctx || batch <= 0 || kv_heads <= 0 || q_heads <= 0 || q_heads % kv_heads || q_heads / kv_heads > TQ_MAX_GROUPS || n_nodes <= 0 || tree_start < 0) return 0;
    return plan(ctx, batch, q_heads, kv_heads, n_nodes, tree_start).bytes;
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
    if (((uintptr_t)lengths & 3) || ((uintptr_t)tree_mask & 7) || ((uintptr_t)workspace & 15)) return TQ_ERR_ARG;
    if (n_nodes == 0) return TQ_OK;
    const Plan p = plan(ctx, cache->batch, q_heads, cache->kv_heads, n_nodes, tree_start);
    const int64_t n_rows = p.n_tiles * p.rows;
    if (n_rows / 8 >= 0x7fffffff) return TQ_ERR_UNSUPPORTED;
    if (!workspace || workspace_bytes < p.bytes) return TQ_ERR_WORKSPACE;
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    TreeArgs a = {};
    a.k_codes = cache->k_codes, a.k_norms = cache->k_norms, a.k_signs = cache->k_signs, a.k_rnorms = cache->k_rnorms;
    a.v_codes = cache->v_codes, a.v_norms = cache->v_norms, a.cache_sb = cache->stride_b, a.cache_sh = cache->stride_h, a.capacity = cache->capacity;
    a.batch = cache->batch, a.kv_heads = cache->kv_heads, a.group = q_heads / cache->kv_heads, a.nodes = n_nodes, a.tree_start = tree_start;
    a.positions = p.positions, a.tiles = p.tiles, a.rows = p.rows, a.ctas = p.ctas;
    a.seq_start = cache->seq_start, a.lengths = lengths, a.mask = tree_mask;
    a.image_k = ctx->img_rot_k.data, a.image_s = ctx->img_qjl.data, a.image_v = ctx->img_rot_v.data;
    a.unscale_k = kUmmaRestore * ctx->img_rot_k.unscale, a.unscale_s = kUmmaRestore * ctx->img_qjl.unscale, a.unscale_v = kUmmaRestore * ctx->img_rot_v.unscale / (ctx->cen_v_scale * 0x1p-14f);
    a.centers_k = ctx->centers_k, a.centers_v = ctx->centers_v, a.cen_v_scale = ctx->cen_v_scale * 0x1p-14f;
    a.q = q->data, a.qb = q->stride_b, a.qh = q->stride_h, a.qt = q->stride_t;
    a.out = const_cast<void *>(out->data), a.ob = out->stride_b, a.oh = out->stride_h, a.ot = out->stride_t;
    a.qop = reinterpret_cast<uint4 *>(ws + p.qop);
    a.part_ml = reinterpret_cast<float *>(ws + p.ml), a.part_o = reinterpret_cast<float4 *>(ws + p.o);
    a.error_flag = ctx->error_flag;
    TQ_CUDA_CHECK(q->dtype == TQ_DTYPE_F16 ? launch<__half>(a, ctx, n_rows, (cudaStream_t)stream)
                                           : launch<__nv_bfloat16>(a, ctx, n_rows, (cudaStream_t)stream));
    return TQ_OK;
}
