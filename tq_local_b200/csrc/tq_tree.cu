// Attention of drafted tokens over the packed cache, on the 5th-generation tensor cores.  The T drafted tokens of every batch entry are
// packed at tokens [tree_start, tree_start + T); node i attends the entry's history [seq_start, length) and the drafted tokens that its
// mask names:
//
//   logit_ij = scale (kn_j c_k[codes_j] . (R_k q_i) + rn_j sqrt(pi/2)/D signs_j . (S q_i)),   out_i = R_v^T sum_j p_ij vn_j c_v[codes_j]
//
// Three launches.  The first rotates and projects the queries, rounds them to fp16 (the scale to base 2 and the sketch's factor folded in)
// and sums up how many blocks of 128 tokens the batch entries have.  The second attends: the 128 rows of a tile are (node, head of the group)
// pairs, its blocks are those of history and drafted tokens laid end to end, and all tiles' blocks laid end to end are cut into
// equal pieces, one a CTA (one CTA an SM).  The third joins a tile's pieces, un-rotates and rounds.
//
// Roles of the second: warps 4-11 turn packed tokens into fp16 operands in shared memory, two threads a token: centres times norm by a
// table of centre pairs in shared memory, +-rn for the signs.  Warp 12 issues the products, S = [Rq | Sq] [K | signs]^T with the queries in TMEM
// and O += P V.  Warps 0-3 take the softmax, a row a thread; the weights go back over S as 16-bit pairs.
// TMEM: S of two blocks, O, the queries, 128 columns each.
#include <math.h>

#include <type_traits>

#include "tq_attn_tc.cuh"
#include "tq_step_blocks.cuh"

namespace {

constexpr int kSoftmaxWarps = 4, kOperandWarps = 16;  // and four more, of which one issues the products
constexpr int kThreads = 32 * (kSoftmaxWarps + kOperandWarps + 4);
constexpr int kBlock = 128;  // tokens of a block

struct TreeArgs {
    const uint8_t *k_codes, *k_signs, *v_codes;
    const uint16_t *k_norms, *k_rnorms, *v_norms;
    int64_t cache_sb, cache_sh;
    int batch, kv_heads, group, nodes, tree_start;
    int positions, tiles, rows;  // nodes of a tile, tiles of a (batch entry, KV head), rows of a tile that hold something
    const int *seq_start, *lengths;
    const uint64_t *mask;
    const uint16_t *image_k, *image_s, *image_v;  // R_k, S, R_v
    float unscale_k, unscale_s, unscale_v;
    const float *centers_k, *centers_v;
    const void *q;
    void *out;
    int64_t qb, qh, qt, ob, oh, ot;
    int64_t *prefix;  // [batch + 1] blocks of the entries before
    uint16_t *qop;    // [batch][kv_heads][tiles][rows][128 or 256] fp16
    float *part_ml, *part_o;  // [piece][rows][2], [piece][rows][128]
    int ctas;
    int *error_flag;
};

// Where a coordinate lies in the operands and in O: the second and third eight of the last two quarters change places (see the stores below).
__device__ __forceinline__ int turned(int quarter, int eight) { return eight ^ (quarter & 2); }

struct Entry {
    int start, history;
};
__device__ __forceinline__ Entry entry_of(const TreeArgs &a, int b) {
    const int length = a.lengths ? min(max(a.lengths[b], 0), a.tree_start) : a.tree_start;
    const int start = a.seq_start ? min(max(a.seq_start[b], 0), length) : 0;
    return {start, length - start};
}
// tokens that tile t of an entry may see, in blocks
__device__ __forceinline__ int tile_blocks(const TreeArgs &a, int history, int t) {
    const int drafted = a.mask ? a.nodes : min(a.nodes, (t + 1) * a.positions);
    return (history + drafted + kBlock - 1) / kBlock;
}
__device__ __forceinline__ int head_blocks(const TreeArgs &a, int history) {
    int n = 0;
    for (int t = 0; t < a.tiles; ++t) n += tile_blocks(a, history, t);
    return n;
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

// TMEM and the barriers of such a kernel, and its product: the rows are in TMEM as hi and lo terms at +256 and +320, the sums come at +128 i.
struct RowTile {
    uint32_t tmem, bar_image, bar_mma;
    bool lost = false;
    __device__ __forceinline__ void start(uint32_t *s_tmem, uint64_t *s_bars, uint32_t images, const uint16_t *image0, const uint16_t *image1) {
        bar_image = smem_u32(s_bars), bar_mma = bar_image + 8;
        if (threadIdx.x < 32) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(s_tmem)), "r"(512));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n");
        }
        if (threadIdx.x == 32) {
            mbar_init(bar_image, image1 ? 2 : 1), mbar_init(bar_mma, 1);
            asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            umma_load_image(images, image0, bar_image);
            if (image1) umma_load_image(images + kUmmaImageBytes, image1, bar_image);
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
    template <bool TRANSPOSED> __device__ __forceinline__ void multiply(uint32_t images, int n) {
        if (threadIdx.x < 32 && elect_one()) {
            umma_fence_after();
            if (!mbar_wait(bar_image, 0)) lost = true;
            for (int i = 0; i < n; ++i) umma_issue<2, TRANSPOSED>(tmem + 128 * i, tmem + 256, tmem + 320, images + i * kUmmaImageBytes);
            umma_commit(bar_mma);
        }
        __syncwarp();
        if (!mbar_wait(bar_mma, 0)) lost = true;
        __syncwarp();
        umma_fence_after();
    }
    __device__ __forceinline__ void finish(int *error_flag) {
        if (lost) atomicExch(error_flag, 8);
        umma_fence_before();
        __syncthreads();
        if (threadIdx.x < 32) {
            umma_fence_after();
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512));
        }
    }
};

// Operand rows [Rq | Sq].  Sketch coordinates lie in the order in which the operand's signs do, (i, i + 16) of 32 side by side.
template <typename T, bool QJL> __global__ void __launch_bounds__(kRowThreads, 1) tq_tree_prep_kernel(const __grid_constant__ TreeArgs a, int64_t n_rows, int per_cta) {
    constexpr int kWide = QJL ? 256 : 128;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t s_bars[2];
    __shared__ uint32_t s_tmem;
    const uint32_t images = (smem_u32(smem_raw) + 1023u) & ~1023u;
    tq_launch_dependents();
    RowTile tile;
    tile.start(&s_tmem, s_bars, images, a.image_k, QJL ? a.image_s : nullptr);
    if (blockIdx.x == 0 && threadIdx.x >= kRowThreads - 32) {  // (rows of the last warp are few, or there are many other blocks)
        const int lane = threadIdx.x & 31;
        int64_t before = 0;
        for (int b0 = 0; b0 < a.batch; b0 += 32) {
            const int b = b0 + lane;
            int64_t n = b < a.batch ? (int64_t)head_blocks(a, entry_of(a, b).history) * a.kv_heads : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t x = __shfl_up_sync(0xffffffffu, n, o);
                if (lane >= o) n += x;
            }
            if (b < a.batch) a.prefix[b + 1] = before + n;
            before += __shfl_sync(0xffffffffu, n, 31);
        }
        if (lane == 0) a.prefix[0] = 0;
    }
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
    tile.multiply<false>(images, QJL ? 2 : 1);
#pragma unroll
    for (int i = 0; i < (QJL ? 2 : 1); ++i) {
        const float f = i ? a.unscale_s * (1.2533141373155003f / (float)TQ_D) : a.unscale_k;
        uint32_t y[32], o[16];
        __syncwarp();
        tmem_ld32(tile.tmem + 128 * i + lanes + 32 * part, y);
        tmem_ld_wait(y);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int lo = i ? e : 2 * e, hi = i ? e + 16 : 2 * e + 1;
            o[e] = half2_bits(__uint_as_float(y[lo]) * f, __uint_as_float(y[hi]) * f);
        }
        if (mine) {
            uint4 *dst = reinterpret_cast<uint4 *>(a.qop + r * kWide + 128 * i + 32 * part);
#pragma unroll
            for (int e = 0; e < 4; ++e) dst[turned(part, e)] = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
        }
    }
    tile.finish(a.error_flag);
}

// ---------------------------------------------------------------------------------------------------- attention
// Shared memory: two stages of keys and of values, one of signs, and the tables of centre pairs.  A slot of a table holds its pair once per
// lane, so that every lane reads its own bank.
template <int KB, int VB, bool QJL> struct Layout {
    static constexpr int kKeys = 0, kValues = 2 * kUmmaTermBytes, kSigns = 4 * kUmmaTermBytes;
    static constexpr int kKeyTable = kSigns + (QJL ? kUmmaTermBytes : 0), kValueTable = kKeyTable + 128 * (1 << 2 * KB);
    static constexpr int kBytes = kValueTable + 128 * (1 << 2 * VB) + 1024;
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

// Bits [base, base + 32) of what a row sees, base relative to the first drafted token: all of the history, then the mask.
__device__ __forceinline__ uint32_t seen_word(uint64_t mask, int chain_end, int base) {
    uint32_t r = 0;
    if (base < 0) r = base <= -32 ? 0xffffffffu : (1u << -base) - 1u;
    if (chain_end >= 0) {  // a chain: nodes [0, chain_end)
        const int n = chain_end - base;
        return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : r | ((1u << n) - 1u);
    }
    if (base <= -32 || base >= 64) return r;
    return r | (uint32_t)(base < 0 ? mask << -base : mask >> base);
}

template <int KB, int VB, bool QJL> __global__ void __launch_bounds__(kThreads, 1) tq_tree_kernel(const __grid_constant__ TreeArgs a) {
    using L = Layout<KB, VB, QJL>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t s_bars[2 + 2 + 2 + 2 + 2 + 1 + 1];
    __shared__ uint32_t s_tmem;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t bars = smem_u32(s_bars);
    // full: operands are there; kfree, vfree: the products that read keys and signs, or values, are done; s: logits are there; p: weights are there;
    // o: O += P V is done; q: queries are there
    const uint32_t bar_full = bars, bar_kfree = bars + 16, bar_vfree = bars + 32, bar_s = bars + 48, bar_p = bars + 64, bar_o = bars + 80, bar_q = bars + 88;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    constexpr int kProducts = kSoftmaxWarps + kOperandWarps;
    const int row_warps = (a.rows + 31) >> 5;  // warps of the softmax that have rows (the others' rows of S and O are what they are)
    if (warp == kProducts) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&s_tmem)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n");
    }
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar_full + 8 * i, 16 * kOperandWarps), mbar_init(bar_kfree + 8 * i, 1), mbar_init(bar_vfree + 8 * i, 1);
            mbar_init(bar_s + 8 * i, 1), mbar_init(bar_p + 8 * i, 32 * row_warps);
        }
        mbar_init(bar_o, 1), mbar_init(bar_q, 32 * row_warps);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    {
        const float ck = a.centers_k[lane & 15], cv = a.centers_v[lane & 15];
        auto fill = [&](uint32_t table, int bits, float centre) {
            for (int e = warp; e < 1 << 2 * bits; e += kThreads / 32) {
                const float lo = __shfl_sync(0xffffffffu, centre, e & ((1 << bits) - 1)), hi = __shfl_sync(0xffffffffu, centre, e >> bits);
                asm volatile("st.shared.u32 [%0], %1;\n" ::"r"(table + 128 * e + 4 * lane), "r"(half2_bits(lo, hi)) : "memory");
            }
        };
        fill(base + L::kKeyTable, KB, ck);
        fill(base + L::kValueTable, VB, cv);
    }
    umma_fence_before();
    __syncthreads();
    umma_fence_after();
    tq_grid_dependency_wait();
    tq_launch_dependents();
    const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0), t_o = tmem + 256, t_q = tmem + 384;

    // ---- this CTA's blocks: [flat, flat_end) of all tiles' blocks laid end to end
    const int64_t total = a.prefix[a.batch], chunk = (total + a.ctas - 1) / a.ctas;
    int64_t flat = (int64_t)blockIdx.x * chunk;
    const int64_t flat_end = min(flat + chunk, total);
    struct Segment {  // the part of one tile inside this CTA's piece: blocks [k, k_end)
        int b, h, t, history, start, k, k_end;
        int64_t tile;
    };
    int b_at = 0;  // the entry that holds block `flat`
    if (flat < flat_end)
        for (int b0 = 0, n = 32; n == 32; b0 += 32) {
            const int64_t end = a.prefix[min(b0 + lane + 1, a.batch)];
            n = __popc(__ballot_sync(0xffffffffu, b0 + lane < a.batch && end <= flat));
            b_at += n;
        }
    int64_t b_first = flat < flat_end ? a.prefix[b_at] : 0, b_next = flat < flat_end ? a.prefix[b_at + 1] : 0;
    auto next_segment = [&]() {
        while (flat >= b_next) ++b_at, b_first = b_next, b_next = a.prefix[b_at + 1];
        Segment g;
        const Entry e = entry_of(a, b_at);
        const int per_head = head_blocks(a, e.history);
        int in = (int)(flat - b_first);
        g.b = b_at, g.h = in / per_head, in -= g.h * per_head, g.start = e.start, g.history = e.history;
        int nb = tile_blocks(a, e.history, 0);
        for (g.t = 0; in >= nb;) in -= nb, ++g.t, nb = tile_blocks(a, e.history, g.t);
        g.k = in;
        const int64_t left = flat_end - flat;
        g.k_end = left < nb - in ? in + (int)left : nb;
        g.tile = ((int64_t)g.b * a.kv_heads + g.h) * a.tiles + g.t;
        flat += g.k_end - g.k;
        return g;
    };
    bool lost = false;  // a wait of this thread ran out: it waits for nothing more
    auto wait = [&](uint32_t bar, uint32_t parity) {
        if (!lost && !mbar_wait(bar, parity)) lost = true;
    };

    if (warp >= kProducts) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;\n");
        if (warp == kProducts && elect_one()) {
            // ---------------- products, by one thread; n counts blocks since the kernel began
            constexpr uint32_t instr_s = umma_instr<false>(), instr_o = umma_instr<true>();
            auto scores = [&](uint32_t n) {
                wait(bar_full + 8 * (n & 1), n >> 1 & 1);
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
                    wait(bar_p + 8 * (n & 1), n >> 1 & 1);
                    umma_fence_after();
                    attn_values(t_o, tmem + 128 * (n & 1), base + L::kValues + (n & 1) * kUmmaTermBytes, instr_o, !first);
                    umma_commit(bar_vfree + 8 * (n & 1));
                    umma_commit(bar_o);
                }
            }
        }
    } else if (warp >= kSoftmaxWarps) {
        // ---------------- operands.  Half of the warps take the even blocks, half the odd ones: a thread's loads have two blocks' time to arrive, and
        // none are on their way when it fences its stores (the fence would wait for them).  A quarter of two tokens' coordinates a thread, four
        // lanes to a token, so that a load covers whole lines.
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;\n");
        const uint32_t half = (uint32_t)(warp - kSoftmaxWarps) / (kOperandWarps / 2);
        const int quarter = lane & 3, row0 = 16 * ((warp - kSoftmaxWarps) % (kOperandWarps / 2)) + (lane >> 2);  // and row0 + 8
        uint32_t kw[2][KB + 1] = {}, vw[2][VB + 1] = {}, sw[2] = {};
        uint16_t kn[2], vn[2], rn[2];
        Segment g;
        int k = 0, k_end = 0;
        uint32_t n = 0;  // blocks since the kernel began
        auto words = [&](const uint8_t *src, auto count, uint32_t *w) {
            constexpr int n = decltype(count)::value;
            if constexpr (n == 4) {
                const uint4 x = __ldg(reinterpret_cast<const uint4 *>(src));
                w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
            } else if constexpr (n == 2) {
                const uint2 x = __ldg(reinterpret_cast<const uint2 *>(src));
                w[0] = x.x, w[1] = x.y;
            } else {
#pragma unroll
                for (int i = 0; i < n; ++i) w[i] = __ldg(reinterpret_cast<const uint32_t *>(src) + i);
            }
        };
        auto next_block = [&]() {  // false behind the last
            if (k == k_end) {
                if (flat >= flat_end) return false;
                g = next_segment(), k = g.k, k_end = g.k_end;
            }
            return true;
        };
        auto fetch = [&]() {  // the block's tokens of this thread
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int v = k * kBlock + row0 + 8 * i;
                kn[i] = vn[i] = rn[i] = 0;
                if (v < g.history + a.nodes) {
                    const int64_t t = g.b * a.cache_sb + g.h * a.cache_sh + (v < g.history ? g.start + v : a.tree_start + v - g.history);
                    words(a.k_codes + t * 16 * KB + 4 * KB * quarter, std::integral_constant<int, KB>(), kw[i]);
                    words(a.v_codes + t * 16 * VB + 4 * VB * quarter, std::integral_constant<int, VB>(), vw[i]);
                    kn[i] = __ldg(a.k_norms + t), vn[i] = __ldg(a.v_norms + t);
                    if (QJL) sw[i] = __ldg(reinterpret_cast<const uint32_t *>(a.k_signs + t * 16) + quarter), rn[i] = __ldg(a.k_rnorms + t);
                }
            }
        };
        const uint32_t lane_k = base + L::kKeyTable + 4 * lane, lane_v = base + L::kValueTable + 4 * lane;
        // Eight lanes store two tokens' quarters: with the last two quarters' eights turned, to eight different banks of 16 bytes.
        const uint32_t turn = (quarter & 1) * 4 ^ (quarter & 2) ^ (row0 & 7), stage = half * kUmmaTermBytes;
        const uint32_t my_row = base + (quarter >> 1) * kUmmaSlabBytes + (row0 >> 3) * 1024 + (row0 & 7) * 128;
        auto put = [&](uint32_t at, auto word) {  // word(i, j): word j of the 16 of token i
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    sts128(my_row + at + 1024 * i + ((c ^ turn) << 4), word(i, 4 * c), word(i, 4 * c + 1), word(i, 4 * c + 2), word(i, 4 * c + 3));
        };
        for (; next_block(); ++n, ++k) {
            if ((n & 1) != half) continue;
            fetch();
            if (n > 1) wait(bar_vfree + 8 * half, (n >> 1 & 1) ^ 1);  // (two blocks ago; its logits came before)
            put(L::kKeys + stage, [&](int i, int j) { return centre_pair<KB>(kw[i], j, lane_k, kn[i] * 0x10001u); });
            put(L::kValues + stage, [&](int i, int j) { return centre_pair<VB>(vw[i], j, lane_v, vn[i] * 0x10001u); });
            if (QJL) {
                if (n) wait(bar_kfree + 8 * (half ^ 1), (n - 1) >> 1 & 1);  // (the signs have one stage)
                put(L::kSigns, [&](int i, int j) {  // signs j and j + 16 of a word; a set bit is +
                    return ((sw[i] << (15 - j)) & 0x80008000u) ^ (rn[i] * 0x10001u) ^ 0x80008000u;
                });
            }
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            mbar_arrive_one(bar_full + 8 * half);
        }
    } else {
        // ---------------- softmax, one row a thread
        asm volatile("setmaxnreg.inc.sync.aligned.u32 168;\n");
        const int row = tid;
        const uint32_t lanes = (uint32_t)(warp * 32) << 16;
        constexpr int kWide = QJL ? 256 : 128;
        uint32_t n = 0;
        if (warp < row_warps) while (flat < flat_end) {
            const Segment g = next_segment();
            const int node = g.t * a.positions + row / a.group;
            const bool live = row < a.rows && node < a.nodes;
            const uint64_t mask = live && a.mask ? a.mask[(int64_t)g.b * a.nodes + node] & (~0ull >> (64 - a.nodes)) : 0;
            const int chain_end = a.mask ? -1 : live ? node + 1 : 0;
            // ---- the queries (the products that read the ones before are done: their logits were here)
            const uint4 *src = reinterpret_cast<const uint4 *>(a.qop + (g.tile * a.rows + row) * kWide);
#pragma unroll
            for (int i = 0; i < kWide / 64; ++i) {
                uint32_t r[32];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint4 x = row < a.rows ? src[8 * i + e] : make_uint4(0, 0, 0, 0);
                    r[4 * e] = x.x, r[4 * e + 1] = x.y, r[4 * e + 2] = x.z, r[4 * e + 3] = x.w;
                }
                __syncwarp();
                tmem_st32(t_q + lanes + 32 * i, r);
            }
            tmem_st_wait();
            umma_fence_before();
            mbar_arrive_one(bar_q);
            float m_ref = -INFINITY;
            uint64_t sum[2] = {0, 0};
            for (int k = g.k; k < g.k_end; ++k, ++n) {
                const uint32_t t_s = tmem + 128 * (n & 1) + lanes;
                wait(bar_s + 8 * (n & 1), n >> 1 & 1);
                __syncwarp();
                umma_fence_after();
                uint32_t s[128];
#pragma unroll
                for (int i = 0; i < 4; ++i) tmem_ld32(t_s + 32 * i, s + 32 * i);
#pragma unroll
                for (int i = 0; i < 4; ++i) tmem_ld_wait(s + 32 * i);
                if ((k + 1) * kBlock > g.history) {
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const uint32_t seen = seen_word(mask, chain_end, k * kBlock + 32 * x - g.history);
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (!(seen >> i & 1)) s[32 * x + i] = 0xff800000u;
                    }
                }
                float top[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) top[i] = max3(__uint_as_float(s[i]), __uint_as_float(s[i + 4]), __uint_as_float(s[i + 8]));
#pragma unroll
                for (int i = 12; i < 124; i += 8)
#pragma unroll
                    for (int e = 0; e < 4; ++e) top[e] = max3(top[e], __uint_as_float(s[i + e]), __uint_as_float(s[i + e + 4]));
                float peak = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                peak = fmaxf(peak, max3(__uint_as_float(s[124]), __uint_as_float(s[125]), fmaxf(__uint_as_float(s[126]), __uint_as_float(s[127]))));
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
                            uint32_t o[32];
                            tmem_ld32(t_o + lanes + 32 * i, o);
                            tmem_ld_wait(o);
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                            tmem_st32(t_o + lanes + 32 * i, o);
                        }
                    }
                }
                const float shift = m_ref == -INFINITY ? 0.f : -m_ref;
                const uint64_t shift2 = f32x2(shift, shift);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t p[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        float x, y;
                        f32x2_split(f32x2_add(f32x2(__uint_as_float(s[64 * half + 2 * i]), __uint_as_float(s[64 * half + 2 * i + 1])), shift2), x, y);
                        x = exp2_hw(x), y = exp2_hw(y);
                        sum[i & 1] = f32x2_add(sum[i & 1], f32x2(x, y));
                        p[i] = pack16<false>(x, y);
                    }
                    tmem_st32(t_s + 32 * half, p);
                }
                tmem_st_wait();
                umma_fence_before();
                // (the wait for the last values tells them from those before only if these are known to be done)
                if (k > g.k && k + 1 == g.k_end) wait(bar_o, (n - 1) & 1);
                mbar_arrive_one(bar_p + 8 * (n & 1));
            }
            // ---- this piece of the tile's rows
            float l0, l1;
            f32x2_split(f32x2_add(sum[0], sum[1]), l0, l1);
            wait(bar_o, (n - 1) & 1);
            __syncwarp();
            umma_fence_after();
            const int64_t r = (g.tile + blockIdx.x) * a.rows + row;
            if (live) *reinterpret_cast<float2 *>(a.part_ml + 2 * r) = make_float2(m_ref, l0 + l1);
#pragma unroll 1
            for (int i = 0; i < 4; ++i) {
                uint32_t o[32];
                __syncwarp();
                tmem_ld32(t_o + lanes + 32 * i, o);
                tmem_ld_wait(o);
                if (live)
#pragma unroll
                    for (int e = 0; e < 32; e += 4) *reinterpret_cast<uint4 *>(a.part_o + r * TQ_D + 32 * i + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            }
            umma_fence_before();
        }
    }
    if (lost) atomicExch(a.error_flag, 8);
    umma_fence_before();
    __syncthreads();
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
    const uint32_t images = (smem_u32(smem_raw) + 1023u) & ~1023u;
    float4 *const s_part = reinterpret_cast<float4 *>(smem_raw + (images - smem_u32(smem_raw)) + kUmmaImageBytes);  // [slot][33]
    RowTile tile;
    tile.start(&s_tmem, s_bars, images, a.image_v, nullptr);
    const int slot = threadIdx.x & 127, part = threadIdx.x >> 7;
    const uint32_t lanes = (uint32_t)(threadIdx.x & 96) << 16;
    int rows = 8;
    while (rows < per_cta) rows *= 2;
    const int groups = kUmmaRows / rows, row = slot & (rows - 1), group = slot / rows;
    const int64_t r = (int64_t)blockIdx.x * per_cta + row;
    RowPlace p = {};
    if (row < per_cta && r < n_rows) p = place_of(a, r, n_rows);
    tq_grid_dependency_wait();
    float o[32] = {};
    float m = -INFINITY, l = 0.f;
    if (p.live) {
        const int64_t total = a.prefix[a.batch], chunk = (total + a.ctas - 1) / a.ctas;
        const int history = entry_of(a, p.b).history, t = (int)(p.tile % a.tiles);
        int64_t first = a.prefix[p.b] + (int64_t)p.h * head_blocks(a, history);
        for (int x = 0; x < t; ++x) first += tile_blocks(a, history, x);
        const int64_t c0 = first / chunk, c1 = (first + tile_blocks(a, history, t) - 1) / chunk;
        const int64_t piece0 = (p.tile + c0) * a.rows + p.in;
        const int n = (int)(c1 - c0) + 1;
        const float2 *ml = reinterpret_cast<const float2 *>(a.part_ml) + piece0;
#pragma unroll 4
        for (int c = group; c < n; c += groups) m = fmaxf(m, ml[(int64_t)c * a.rows].x);
#pragma unroll 2
        for (int c = group; c < n; c += groups) {
            const float2 x = ml[(int64_t)c * a.rows];
            const float4 *src = reinterpret_cast<const float4 *>(a.part_o + (piece0 + (int64_t)c * a.rows) * TQ_D + 32 * part);
            const float f = x.y == 0.f ? 0.f : exp2f(x.x - m);  // (a piece in which the row saw nothing)
            l += f * x.y;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float4 v = src[2 * turned(part, i >> 1) + (i & 1)];
                o[4 * i] += f * v.x, o[4 * i + 1] += f * v.y, o[4 * i + 2] += f * v.z, o[4 * i + 3] += f * v.w;
            }
        }
    }
    if (groups > 1) {
        if (part == 0) s_ml[slot] = make_float2(m, l);
#pragma unroll
        for (int i = 0; i < 8; ++i) s_part[slot * 33 + 8 * part + i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        __syncthreads();
        l = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = 0.f;
        if (p.live && group == 0) {
            m = -INFINITY;
            for (int x = 0; x < groups; ++x) m = fmaxf(m, s_ml[x * rows + row].x);
            for (int x = 0; x < groups; ++x) {
                const float2 ml = s_ml[x * rows + row];
                const float f = ml.y == 0.f ? 0.f : exp2f(ml.x - m);
                l += f * ml.y;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float4 v = s_part[(x * rows + row) * 33 + 8 * part + i];
                    o[4 * i] += f * v.x, o[4 * i + 1] += f * v.y, o[4 * i + 2] += f * v.z, o[4 * i + 3] += f * v.w;
                }
            }
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
    tile.multiply<true>(images, 1);
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
    size_t prefix, qop, ml, o, bytes;  // workspace offsets
};
Plan plan(const tq_ctx *ctx, int64_t batch, int q_heads, int kv_heads, int nodes, int tree_start) {
    Plan p;
    const int group = q_heads / kv_heads;
    p.positions = kUmmaRows / group;
    p.tiles = (nodes + p.positions - 1) / p.positions;
    p.rows = (nodes < p.positions ? nodes : p.positions) * group;
    p.n_tiles = batch * kv_heads * p.tiles;
    const int64_t most = p.n_tiles * (((int64_t)tree_start + nodes + kBlock - 1) / kBlock);
    p.ctas = most < ctx->sm_count ? (int)most : ctx->sm_count;
    auto take = [at = (size_t)0](size_t bytes) mutable {
        const size_t r = at;
        at += (bytes + 255) / 256 * 256;
        return r;
    };
    const size_t pieces = (size_t)(p.n_tiles + p.ctas) * p.rows;
    p.prefix = take((batch + 1) * sizeof(int64_t));
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
    constexpr int smem = (QJL ? 2 : 1) * kUmmaImageBytes + 1024;
    const cudaError_t e = tq_allow_shared<tq_tree_prep_kernel<T, QJL>>(device, smem);
    return e != cudaSuccess ? e : tq_launch_kernel(tq_tree_prep_kernel<T, QJL>, dim3(blocks), dim3(kRowThreads), smem, stream, false, a, n_rows, per_cta);
}

template <typename T> cudaError_t launch(const TreeArgs &a, const tq_ctx *ctx, int64_t n_rows, cudaStream_t stream) {
    const bool qjl = ctx->use_qjl != 0;
    const int device = ctx->device;
    const int64_t share = ((n_rows + ctx->sm_count - 1) / ctx->sm_count + 7) / 8 * 8;
    const int per_cta = share < kUmmaRows ? (int)share : kUmmaRows;
    const unsigned blocks = (unsigned)((n_rows + per_cta - 1) / per_cta);
    cudaError_t e = qjl ? launch_prep<T, true>(a, n_rows, blocks, per_cta, device, stream) : launch_prep<T, false>(a, n_rows, blocks, per_cta, device, stream);
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
    a.v_codes = cache->v_codes, a.v_norms = cache->v_norms, a.cache_sb = cache->stride_b, a.cache_sh = cache->stride_h;
    a.batch = cache->batch, a.kv_heads = cache->kv_heads, a.group = q_heads / cache->kv_heads, a.nodes = n_nodes, a.tree_start = tree_start;
    a.positions = p.positions, a.tiles = p.tiles, a.rows = p.rows, a.ctas = p.ctas;
    a.seq_start = cache->seq_start, a.lengths = lengths, a.mask = tree_mask;
    a.image_k = ctx->img_rot_k.data, a.image_s = ctx->img_qjl.data, a.image_v = ctx->img_rot_v.data;
    a.unscale_k = kUmmaRestore * ctx->img_rot_k.unscale, a.unscale_s = kUmmaRestore * ctx->img_qjl.unscale, a.unscale_v = kUmmaRestore * ctx->img_rot_v.unscale;
    a.centers_k = ctx->centers_k, a.centers_v = ctx->centers_v;
    a.q = q->data, a.qb = q->stride_b, a.qh = q->stride_h, a.qt = q->stride_t;
    a.out = const_cast<void *>(out->data), a.ob = out->stride_b, a.oh = out->stride_h, a.ot = out->stride_t;
    a.prefix = reinterpret_cast<int64_t *>(ws + p.prefix), a.qop = reinterpret_cast<uint16_t *>(ws + p.qop);
    a.part_ml = reinterpret_cast<float *>(ws + p.ml), a.part_o = reinterpret_cast<float *>(ws + p.o);
    a.error_flag = ctx->error_flag;
    TQ_CUDA_CHECK(q->dtype == TQ_DTYPE_F16 ? launch<__half>(a, ctx, n_rows, (cudaStream_t)stream)
                                           : launch<__nv_bfloat16>(a, ctx, n_rows, (cudaStream_t)stream));
    return TQ_OK;
}
