// Attention of a whole prompt over dense keys and values on the 5th-generation tensor cores:
//
//   out_i = sum_j softmax_j(scale q_i . k_j) v_j  over the keys a query sees
//
// in one pass over the keys, 128 at a time, with the running maximum and sum of the softmax; logits and weights stay on the SM.
//
// Rows.  The query heads of a KV head share its keys, so a tile's 128 rows are (position, head of the group) pairs, positions
// outermost: keys and values are read once for all of them, and a tile ends at its own last position, which leaves little of a
// causal mask inside it.  A CTA owns two tiles (one, where tiles are few): while the tensor core multiplies for one, the other's
// warps take exponentials.
//
// Roles.  Warps 0-3 and 4-7: the softmax of a tile each, one row a thread.  Warp 8: requests the query tiles and the key and value blocks
// (tensor maps, 128-byte swizzle, a ring of 32 KB slots).  Warps 9 and 10: issue the products of a tile each.  Warp 11: clears values that
// are outside the sequence.  S = Q K^T with both operands in shared memory; the weights go back to TMEM over S as 16-bit pairs and are the A
// operand of O += P V.  TMEM: S of the two tiles, O of the two tiles, 128 columns each.
//
// What bounds it: 32768 tokens, 32 / 8 heads, bf16, take 7.4 ms on a card at rest (1190 TFLOP/s) and 8.4 ms back to back, where the card's
// power limit lowers its clock (1050; the library's matrix product falls from 1657 to 1376).  Between steps the tensor core waits for exponentials
// (16 a clock and SM against 8192 operations: as long as the products) and for the hand-over of logits and weights.
#include <cuda.h>
#include <math.h>

#include <type_traits>

#include "tq_attn_tc.cuh"

namespace {

__device__ int g_prompt_status;

constexpr int kSoftmax = 256;                    // threads: a row of two tiles each
constexpr int kThreads = kSoftmax + 128;
constexpr int kBlock = 128;                      // keys of a block
// Keys of a step.  The logits of a tile have 128 columns of TMEM, and the weights go over them: with 64 keys a step there are two sets, and the
// products for one run while the softmax takes the other (8192 tokens, 32 / 8 heads, bf16: 512 us; 597 with 128 keys and one set).
constexpr int kUnit = 64;
constexpr int kBuffers = kBlock / kUnit;         // steps whose logits are held at a time, and steps of a block
// Pairs of exponentials out of eight that the polynomial takes: none 573 us, one 565, two 563, three 566, four 577 (as above, back to back, where the
// card's power limit holds).
constexpr int kPolyOf8 = 2;
constexpr int kSlotBytes = kUmmaTermBytes;       // 128 rows x 128 16-bit values
constexpr int kSlots = 5;
// two query tiles, the ring, barriers and the TMEM address
constexpr int kBarsAt = (2 + kSlots) * kSlotBytes, kBars = 2 + 4 + 4 + 2 + 2 * kSlots + 3 + 2;
constexpr int kSmem = kBarsAt + 8 * kBars + 16;

struct PromptArgs {
    void *out;
    int64_t ob, oh, ot;
    int batch, kv_heads, group, positions;  // positions of a tile: 128 / group
    int n_q, n_kv, total, n_items, tiles_per_cta, splits;
    const int *seq_start, *cu_seqlens;
    float scale_log2;  // |scale| log2(e)
    bool causal, negate;
    float *part_ml, *part_o;  // splits > 1: [row][split] maximum (log2) and sum, [row][split][128]
};

__device__ __forceinline__ void load_map(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z, int w, int v) {
    asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];\n" ::"r"(dst),
                 "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w), "r"(v)
                 : "memory");
}
__device__ __forceinline__ void load_map(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z, int w) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];\n" ::"r"(dst),
                 "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
                 : "memory");
}

// Sequence b of a packed call: its first token, and how many there are - inside [0, total) and no more than n_q, whatever cu_seqlens holds.
__device__ __forceinline__ int2 sequence_of(const PromptArgs &a, int b) {
    const int first = min(max(a.cu_seqlens[b], 0), a.total);
    return make_int2(first, min(min(a.cu_seqlens[b + 1], a.total) - first, a.n_q));
}

// What a row's sums are multiplied with.  A row that sees no key has zeros.  One whose logits are all -inf has no softmax: NaN (its sum is 0, or some 2^-125
// where exponentials come from the polynomial).
__device__ __forceinline__ float inverse_sum(float m, float l, bool sees) { return !sees ? 0.f : m == -INFINITY ? __int_as_float(0x7fffffff) : 1.f / l; }

template <bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
    tq_prompt_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                     const __grid_constant__ PromptArgs a) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];  // (swizzle atoms need 1024-byte alignment, and there is no room to spare)
    // ---- this CTA's work: the longest tiles come first
    const int h = blockIdx.x % a.kv_heads, b = blockIdx.x / a.kv_heads % a.batch;
    const int item = a.n_items - 1 - blockIdx.x / (a.kv_heads * a.batch);
    int n_q = a.n_q, n_kv = a.n_kv, t0 = 0;
    if (a.cu_seqlens) {
        const int2 seq = sequence_of(a, b);
        t0 = seq.x, n_q = n_kv = seq.y;
    }
    const int first_pos = item * a.tiles_per_cta * a.positions;
    if (first_pos >= n_q) return;
    const int offset = n_kv - n_q;
    const int start = a.seq_start ? min(max(a.seq_start[b], 0), n_kv) : 0;
    const int block0 = start / kBlock;
    auto units_of = [&](int w) {
        const int pos = first_pos + w * a.positions;
        if (w >= a.tiles_per_cta || pos >= n_q) return 0;
        const int end = a.causal ? min(n_kv, min(pos + a.positions, n_q) + offset) : n_kv;
        return end > start ? (end + kUnit - 1) / kUnit - block0 * kBuffers : 0;
    };
    int nu0 = units_of(0), nu1 = units_of(1), first_block = block0;
    if (a.splits > 1) {
        const int share = (max(nu0, nu1) + kBuffers * a.splits - 1) / (kBuffers * a.splits) * kBuffers, lo = share * blockIdx.y;  // (whole blocks)
        first_block += lo / kBuffers, nu0 = min(max(nu0 - lo, 0), share), nu1 = min(max(nu1 - lo, 0), share);
    }
    const int nu = max(nu0, nu1), nb = (nu + kBuffers - 1) / kBuffers;

    const uint32_t base = smem_u32(smem_raw), ring = base + 2 * kSlotBytes, bars = base + kBarsAt;
    uint32_t *const s_tmem = reinterpret_cast<uint32_t *>(smem_raw + kBarsAt + 8 * kBars);
    int *const s_asked = reinterpret_cast<int *>(s_tmem + 1);  // copies that were requested: of keys and values, and of which tiles' queries
    if (base & 1023u) {
        if (threadIdx.x == 0) atomicExch(&g_prompt_status, 2);
        return;
    }
    // q: queries are there; s[tile][unit & 1]: logits are there; p[tile][unit & 1]: weights are there; o[tile]: O += P V is done; full, empty: slots;
    // done[tile]: see the end
    const uint32_t bar_q = bars, bar_s = bars + 16, bar_p = bars + 48, bar_o = bars + 80, bar_full = bars + 96, bar_empty = bar_full + 8 * kSlots, bar_ask = bar_empty + 8 * kSlots, bar_clean = bar_ask + 8, bar_done = bar_clean + 16;
    const int tid = threadIdx.x, warp = tid >> 5;
    if (warp == kSoftmax / 32 + 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(s_tmem)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n");
    }
    // copies: Q0, K0, Q1, V0, K1, V1, ...; the first ones, which wait for no free slot, leave before the CTA has set up the rest
    auto load_q = [&](int w) {
        mbar_expect_tx(bar_q + 8 * w, 256 * a.positions * a.group);
        for (int x = 0; x < 2; ++x)
            load_map(base + w * kSlotBytes + x * kUmmaSlabBytes, &map_q, bar_q + 8 * w, 64 * x, 0, t0 + first_pos + w * a.positions, h, a.cu_seqlens ? 0 : b);
    };
    auto load_slot = [&](int i) {  // keys of block i / 2, or its values
        const int slot = i % kSlots;
        const uint32_t bar = bar_full + 8 * slot;
        mbar_expect_tx(bar, kSlotBytes);
        for (int x = 0; x < 2; ++x)
            load_map(ring + slot * kSlotBytes + x * kUmmaSlabBytes, i & 1 ? &map_v : &map_k, bar, 64 * x, t0 + (first_block + i / 2) * kBlock, h, a.cu_seqlens ? 0 : b);
    };
    if (warp == kSoftmax / 32 && elect_one()) {
        mbar_init(bar_q, 1), mbar_init(bar_q + 8, 1), mbar_init(bar_ask, 1), mbar_init(bar_clean, 1), mbar_init(bar_clean + 8, 1);
        for (int i = 0; i < 4; ++i) mbar_init(bar_s + 8 * i, 1), mbar_init(bar_p + 8 * i, 4);
        for (int w = 0; w < 2; ++w) mbar_init(bar_o + 8 * w, 1), mbar_init(bar_done + 8 * w, 1);
        for (int s = 0; s < kSlots; ++s) mbar_init(bar_full + 8 * s, 1), mbar_init(bar_empty + 8 * s, 2);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
        if (nu0) load_q(0);
        for (int i = 0; i < min(2 * nb, kSlots); ++i) {
            load_slot(i);
            if (i == 0 && nu1) load_q(1);
        }
    }
    __syncwarp();
    umma_fence_before();
    __syncthreads();
    umma_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *s_tmem, 0);
    bool lost = false;  // a wait of this thread ran out: it waits for nothing more
    auto wait = [&](uint32_t bar, uint32_t parity) {
        if (!lost && !mbar_wait(bar, parity)) lost = true;
    };

    auto dirty = [&](int k) { return (first_block + k) * kBlock < start || (first_block + k + 1) * kBlock > n_kv; };

    if (warp >= kSoftmax / 32) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;\n");
        if (warp == kSoftmax / 32) {
            // ---------------- copies
            if (elect_one()) {
                int i = kSlots;
                for (; i < 2 * nb; ++i) {
                    wait(bar_empty + 8 * (i % kSlots), (i / kSlots & 1) ^ 1);
                    if (lost) break;
                    load_slot(i);
                }
                s_asked[0] = min(2 * nb, i), s_asked[1] = (nu0 > 0) | (nu1 > 0) << 1;
            }
        } else if (warp < kSoftmax / 32 + 3) {
            // ---------------- products of tile w.  A wait costs a thread some 200 cycles even when there is nothing to wait for; a warp a tile keeps
            // the tensor core busy with one tile's products meanwhile.
            const int w = warp - (kSoftmax / 32 + 1), mine = w ? nu1 : nu0;
            if (elect_one()) {
                const uint32_t instr_s = attn_instr<BF16, false>(a.negate) - (((kBlock - kUnit) >> 3) << 17), instr_o = attn_instr<BF16, true>();
                auto slot_addr = [&](int i) { return ring + i % kSlots * kSlotBytes; };
                auto wait_full = [&](int i) { wait(bar_full + 8 * (i % kSlots), i / kSlots & 1); };
                constexpr uint32_t kHalf = kUnit * 128;  // bytes of 64 rows in a slab
                auto scores = [&](int u) {               // S[u % kBuffers] = Q K_u^T
                    const uint64_t q = umma_desc<false>(base + w * kSlotBytes), k = umma_desc<false>(slot_addr(2 * (u / kBuffers)) + u % kBuffers * kHalf);
#pragma unroll
                    for (uint32_t s = 0; s < 8; ++s) {
                        const uint32_t step = ((s >> 2) * kUmmaSlabBytes + (s & 3) * 32) >> 4;
                        umma_ss(tmem + 128 * w + kUnit * (u % kBuffers), q + step, k + step, instr_s, s > 0);
                    }
                    umma_commit(bar_s + 16 * w + 8 * (u % kBuffers));
                };
                auto values = [&](int u) {  // O += P[u % kBuffers] V_u
                    const uint64_t v = umma_desc<true>(slot_addr(2 * (u / kBuffers) + 1) + u % kBuffers * kHalf);
#pragma unroll
                    for (uint32_t s = 0; s < kUnit / 16; ++s)
                        umma_f16(tmem + 256 + 128 * w, tmem + 128 * w + kUnit * (u % kBuffers) + 8 * s, v + ((s * 16 * 128) >> 4), instr_o, u > 0 || s > 0);
                    umma_commit(bar_o + 8 * w);
                };
                auto release = [&](int i) {  // (a slot that is filled again; the other tile's thread does the same)
                    if (i + kSlots < 2 * nb) umma_commit(bar_empty + 8 * (i % kSlots));
                };
                if (nb) {
                    wait_full(0);
                    if (mine) wait(bar_q + 8 * w, 0), scores(0);
                    if (kBuffers > 1 && mine > 1) scores(1);
                    release(0);
                }
                for (int k = 0; k < nb; ++k) {
                    wait_full(2 * k + 1);
                    if (dirty(k)) {
                        if (w == 0) mbar_arrive_one(bar_ask);
                        wait(bar_clean + (k ? 8 : 0), 0);
                    }
                    if (k + 1 < nb) wait_full(2 * k + 2);
#pragma unroll
                    for (int e = 0; e < kBuffers; ++e) {
                        const int u = kBuffers * k + e;
                        if (u >= mine) continue;
                        wait(bar_p + 16 * w + 8 * e, k & 1);
                        umma_fence_after();
                        values(u);
                        if (u + kBuffers < mine) scores(u + kBuffers);  // (over the weights that were multiplied just before)
                    }
                    release(2 * k + 1), release(2 * k + 2);
                }
            }
        } else {
            // ---------------- values that no query sees may hold anything, and 0 * inf is not 0: they become 0 (in the first block and the last)
            for (int k = 0, asked = 0; k < nb; ++k) {
                if (!dirty(k)) continue;
                const int slot = (2 * k + 1) % kSlots, j0 = (first_block + k) * kBlock;
                wait(bar_ask, asked++ & 1);
                __syncwarp();
                for (int i = tid & 31; i < kBlock * 16; i += 32) {
                    const int row = i >> 4;
                    if (row < start - j0 || row >= n_kv - j0) sts128(ring + slot * kSlotBytes + (i & 8) / 8 * kUmmaSlabBytes + row * 128 + (i & 7) * 16, 0, 0, 0, 0);
                }
                asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                mbar_arrive_warp(bar_clean + (k ? 8 : 0));
            }
        }
    } else {
        // ---------------- softmax of tile w, one row a thread
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;\n");
        const int w = warp >> 2, row = tid & 127, mine = w ? nu1 : nu0;
        const int pos = first_pos + w * a.positions + row / a.group;
        const bool live = w < a.tiles_per_cta && row < a.positions * a.group && pos < n_q;
        const int limit = a.causal ? min(n_kv, pos + offset + 1) : n_kv;  // keys [start, limit)
        const int tile_limit = a.causal ? min(n_kv, first_pos + w * a.positions + offset + 1) : n_kv;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, t_o = tmem + 256 + 128 * w + lanes;
        const float c = a.scale_log2;
        float m_ref = -INFINITY;
        uint64_t sum[2] = {0, 0};
        for (int u = 0; u < mine; ++u) {
            const int e = u % kBuffers;
            const uint32_t t_s = tmem + 128 * w + kUnit * e + lanes;
            wait(bar_s + 16 * w + 8 * e, u / kBuffers & 1);
            __syncwarp();
            umma_fence_after();
            uint32_t s[kUnit];
#pragma unroll
            for (int i = 0; i < kUnit; i += 32) tmem_ld32(t_s + i, s + i);
#pragma unroll
            for (int i = 0; i < kUnit; i += 32) tmem_ld_wait(s + i);
            const int j0 = first_block * kBlock + u * kUnit;
            const bool masked = j0 < start || j0 + kUnit > tile_limit;
            if (masked) {
                const int lo = start - j0, hi = limit - j0;
#pragma unroll
                for (int i = 0; i < kUnit; ++i)
                    if (i < lo || i >= hi) s[i] = 0xff800000u;
            }
            float top[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) top[i] = max3(__uint_as_float(s[i]), __uint_as_float(s[i + 4]), __uint_as_float(s[i + 8]));
#pragma unroll
            for (int i = 12; i < kUnit - 4; i += 8)
#pragma unroll
                for (int x = 0; x < 4; ++x) top[x] = max3(top[x], __uint_as_float(s[i + x]), __uint_as_float(s[i + x + 4]));
            const float last = max3(__uint_as_float(s[kUnit - 4]), __uint_as_float(s[kUnit - 3]), fmaxf(__uint_as_float(s[kUnit - 2]), __uint_as_float(s[kUnit - 1])));
            const float peak = max3(max3(top[0], top[1], top[2]), top[3], last);
            if (u == 0) {
                m_ref = peak;
            } else {
                const bool raise = live && (peak - m_ref) * c > kLag;
                if (__any_sync(0xffffffffu, raise)) {
                    float keep = 1.f;
                    if (raise) keep = exp2_hw((m_ref - peak) * c), m_ref = peak;
                    const uint64_t keep2 = f32x2(keep, keep);
                    sum[0] = f32x2_mul(sum[0], keep2), sum[1] = f32x2_mul(sum[1], keep2);
                    wait(bar_o + 8 * w, (u - 1) & 1);  // the values of the unit before; those of this one wait for its weights
                    __syncwarp();
                    umma_fence_after();
#pragma unroll 1
                    for (int i = 0; i < 4; ++i) {
                        uint32_t o[32];
                        tmem_ld32(t_o + 32 * i, o);
                        tmem_ld_wait(o);
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                        tmem_st32(t_o + 32 * i, o);
                    }
                }
            }
            const float shift = m_ref == -INFINITY ? 0.f : -m_ref * c;
            const uint64_t c2 = f32x2(c, c), shift2 = f32x2(shift, shift);
            auto weights = [&](auto poly) {
#pragma unroll
                for (int part = 0; part < kUnit; part += 64) {
                    uint32_t p[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const uint64_t x2 = f32x2_fma(f32x2(__uint_as_float(s[part + 2 * i]), __uint_as_float(s[part + 2 * i + 1])), c2, shift2);
                        float x, y;
                        if (decltype(poly)::value && i % 8 < kPolyOf8) {
                            exp2_poly(x2, x, y);
                        } else {
                            f32x2_split(x2, x, y);
                            x = exp2_hw(x), y = exp2_hw(y);
                        }
                        sum[i & 1] = f32x2_add(sum[i & 1], f32x2(x, y));
                        p[i] = pack16<BF16>(x, y);
                    }
                    tmem_st32(t_s + part / 2, p);
                }
            };
            if (masked) weights(std::false_type());  // (a hidden key's weight is 0)
            else weights(std::true_type());
            tmem_st_wait();
            umma_fence_before();
            // (the wait for the last values tells them from those before only if these are known to be done)
            if (u && u + 1 == mine) wait(bar_o + 8 * w, (u - 1) & 1);
            mbar_arrive_warp(bar_p + 16 * w + 8 * e);
        }
        // ---------------- the tile's rows
        float l0, l1;
        f32x2_split(f32x2_add(sum[0], sum[1]), l0, l1);
        const float l = l0 + l1;
        if (mine) {
            wait(bar_o + 8 * w, (mine - 1) & 1);
            __syncwarp();
            umma_fence_after();
        }
        const int head = h * a.group + row % a.group, lane = tid & 31;
        // Rows leave through the tile's query image, which nobody reads any more, sixteen lanes to a row: a warp's 32 rows of 256 bytes, 16-byte
        // pieces turned by the row.
        const uint32_t stage = base + w * kSlotBytes + (warp & 3) * 32 * 256, turn = lane & 15;
        auto copy_rows = [&](uint64_t to) {  // this lane's row goes to `to` (0: nowhere)
            __syncwarp();
#pragma unroll 4
            for (int i = 0; i < 32; i += 2) {
                const int from = i + (lane >> 4);
                const uint64_t row_to = __shfl_sync(0xffffffffu, to, from);
                const uint4 v = lds128(stage + from * 256 + ((lane & 15) ^ (from & 15)) * 16);
                if (row_to) reinterpret_cast<uint4 *>(row_to)[lane & 15] = v;
            }
            __syncwarp();
        };
        if (a.splits > 1) {
            const int64_t r = (((int64_t)b * a.n_q + pos) * (a.kv_heads * a.group) + head) * a.splits + blockIdx.y;
            if (live) a.part_ml[2 * r] = m_ref * c, a.part_ml[2 * r + 1] = l;
            if (mine) {  // (half of the coordinates at a time, the way the finished rows go, see below)
                const uint64_t to = live ? reinterpret_cast<uint64_t>(a.part_o + r * TQ_D) : 0;
#pragma unroll 1
                for (int i = 0; i < 2; ++i) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        uint32_t o[32];
                        __syncwarp();
                        tmem_ld32(t_o + 64 * i + 32 * x, o);
                        tmem_ld_wait(o);
#pragma unroll
                        for (int e = 0; e < 8; ++e) sts128(stage + lane * 256 + ((8 * x + e) ^ turn) * 16, o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                    }
                    copy_rows(to ? to + 256 * i : 0);
                }
            }
        } else {
            const bool any = limit > start;
            const float inv = inverse_sum(m_ref, l, any);
#pragma unroll 1
            for (int i = 0; i < 4; ++i) {
                uint32_t o[32] = {};
                __syncwarp();
                if (mine) {
                    tmem_ld32(t_o + 32 * i, o);
                    tmem_ld_wait(o);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t r[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        r[x] = any ? pack16<BF16>(__uint_as_float(o[8 * e + 2 * x]) * inv, __uint_as_float(o[8 * e + 2 * x + 1]) * inv) : 0u;
                    sts128(stage + lane * 256 + ((4 * i + e) ^ turn) * 16, r[0], r[1], r[2], r[3]);
                }
            }
            const uint64_t dst = reinterpret_cast<uint64_t>(a.out) + 2 * ((a.cu_seqlens ? 0 : b) * a.ob + head * a.oh + (int64_t)(t0 + pos) * a.ot);
            copy_rows(live ? dst : 0);
        }
    }
    umma_fence_before();
    if (__syncthreads_or(lost)) {
        // A thread whose wait ran out waits for nothing more.  What was set going ends before the CTA does all the same: a copy that landed later would land in
        // another's shared memory.
        if (lost) atomicExch(&g_prompt_status, 1);
        if (warp == kSoftmax / 32 && elect_one()) {
            for (int i = max(s_asked[0] - kSlots, 0); i < s_asked[0]; ++i) mbar_wait(bar_full + 8 * (i % kSlots), i / kSlots & 1);
            for (int w = 0; w < 2; ++w)
                if (s_asked[1] >> w & 1) mbar_wait(bar_q + 8 * w, 0);
        } else if (warp > kSoftmax / 32 && warp < kSoftmax / 32 + 3 && elect_one()) {
            const uint32_t bar = bar_done + 8 * (warp - kSoftmax / 32 - 1);
            umma_commit(bar);
            mbar_wait(bar, 0);
        }
        __syncthreads();
    }
    if (warp == kSoftmax / 32 + 1) {
        umma_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512));
    }
}

// A row's partials from its splits: one warp a row.
template <bool BF16> __global__ void __launch_bounds__(128) tq_prompt_join_kernel(const __grid_constant__ PromptArgs a, int64_t rows) {
    const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31, heads = a.kv_heads * a.group;
    if (r >= rows) return;
    const int head = (int)(r % heads), pos = (int)(r / heads % a.n_q), b = (int)(r / heads / a.n_q);
    int n_q = a.n_q, n_kv = a.n_kv, t0 = 0;
    if (a.cu_seqlens) {
        const int2 seq = sequence_of(a, b);
        t0 = seq.x, n_q = n_kv = seq.y;
        if (pos >= n_q) return;
    }
    const float2 *ml = reinterpret_cast<const float2 *>(a.part_ml) + r * a.splits;
    float m = -INFINITY;
    for (int s = 0; s < a.splits; ++s) m = fmaxf(m, ml[s].x);
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < a.splits; ++s) {
        const float2 part = ml[s];
        if (part.y == 0.f) continue;  // (nothing of it was stored)
        const float f = exp2f(part.x - m);
        const float4 v = reinterpret_cast<const float4 *>(a.part_o + (r * a.splits + s) * TQ_D)[lane];
        l += f * part.y;
        o = make_float4(o.x + f * v.x, o.y + f * v.y, o.z + f * v.z, o.w + f * v.w);
    }
    const int start = a.seq_start ? min(max(a.seq_start[b], 0), a.n_kv) : 0;  // (as in the kernel before)
    const int limit = a.causal ? min(n_kv, pos + n_kv - n_q + 1) : n_kv;
    const float inv = inverse_sum(m, l, limit > start);
    uint2 *dst = reinterpret_cast<uint2 *>(reinterpret_cast<uint8_t *>(a.out) + 2 * ((a.cu_seqlens ? 0 : b) * a.ob + head * a.oh + (int64_t)(t0 + pos) * a.ot)) + lane;
    *dst = make_uint2(pack16<BF16>(o.x * inv, o.y * inv), pack16<BF16>(o.z * inv, o.w * inv));
}

bool aligned(const tq_dense_desc *d, int64_t batch, int heads, int64_t tokens) {  // (an axis of one element has no stride of its own)
    const int64_t strides = (batch > 1 ? d->stride_b : 0) | (heads > 1 ? d->stride_h : 0) | (tokens > 1 ? d->stride_t : 0);
    return !(((uintptr_t)d->data | (uintptr_t)(2 * strides)) & 15);
}

int sm_count() {
    int device = 0, n = 0;
    if (cudaGetDevice(&device) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) {
        cudaGetLastError();
        return 148;
    }
    return n;
}

// One tile a CTA or two, and into how many pieces its keys are cut: what takes the least time by three figures.  A block of keys takes a CTA 1.5 us
// with one tile and 2.3 with two (whose products and exponentials go on beside each other), starting and ending one 4, joining pieces 6 (512 queries
// behind 16384 keys, 32 / 8 heads: 197 us with one tile and one piece, 141 as chosen here: two tiles, two pieces).  Under a causal mask a tile sees the keys before
// the queries and half of theirs on average.
// At most 32 pieces: one query behind 32768 keys, 4 / 1 heads, 31.1 us with 16, 23.8 with 32, 24.7 with 64 (behind 131072, 8 / 2 heads, 98, 59 and 45).  Of two
// blocks at least: one query behind 2048 keys, 32 / 8 heads, 12.5 us with one, 12.0 with two, 13.5 with four, behind 1024 11.0, 11.0 and 16.2.
struct Plan {
    int positions, tiles_per_cta, n_items, splits;
};
Plan plan(int64_t batch, int q_heads, int kv_heads, int n_q, int n_kv) {
    Plan best = {};
    const int positions = kUmmaRows / (q_heads / kv_heads), sms = sm_count(), tiles = (n_q + positions - 1) / positions;
    const int blocks = n_kv >= n_q ? (n_kv - n_q / 2 + kBlock - 1) / kBlock : (n_kv + kBlock - 1) / kBlock;
    double least = 0;
    for (int two = 1; two <= 2; ++two) {
        const int items = (tiles + two - 1) / two;
        const int64_t ctas = batch * kv_heads * items;
        for (int splits = 1; splits <= 32 && (splits == 1 || (ctas * splits <= sms && splits <= blocks / 2)); ++splits) {
            const int64_t rounds = (ctas * splits + sms - 1) / sms;
            const double time = rounds * ((blocks + splits - 1) / splits * (two == 2 ? 2.3 : 1.5) + 4.0) + (splits > 1 ? 6.0 : 0.0);
            if (!best.positions || time < least) best = {positions, two, items, splits}, least = time;
        }
    }
    return best;
}

typedef CUresult (*EncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                             const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
    static const EncodeFn fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            p = nullptr;
        }
        return reinterpret_cast<EncodeFn>(p);
    }();
    return fn;
}

// A map of a 16-bit tensor of 128 coordinates with `dims - 1` outer axes, copied in boxes of 64 coordinates.
bool encode(CUtensorMap *map, bool bf16, const void *data, int dims, const int64_t *sizes, const int64_t *strides, const int *box) {
    cuuint64_t size[5] = {TQ_D}, stride[4];
    cuuint32_t boxes[5] = {64}, steps[5] = {1, 1, 1, 1, 1};
    for (int i = 1; i < dims; ++i) {
        size[i] = (cuuint64_t)sizes[i - 1], boxes[i] = (cuuint32_t)box[i - 1];
        stride[i - 1] = sizes[i - 1] > 1 ? (cuuint64_t)strides[i - 1] * 2 : 2 * TQ_D;  // (an axis of one element has no stride of its own)
    }
    const EncodeFn fn = encode_fn();
    return fn && fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, dims, const_cast<void *>(data), size, stride, boxes, steps,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool BF16> int32_t launch(const tq_dense_desc *q, const tq_dense_desc *k, const tq_dense_desc *v, int64_t tokens_q, int64_t tokens_kv, int maps_batch,
                                    const PromptArgs &a, cudaStream_t stream) {
    CUtensorMap maps[3];
    const int64_t q_sizes[4] = {a.group, tokens_q, a.kv_heads, maps_batch}, q_strides[4] = {q->stride_h, q->stride_t, q->stride_h * a.group, q->stride_b};
    const int q_box[4] = {a.group, a.positions, 1, 1}, kv_box[3] = {kBlock, 1, 1};
    bool ok = encode(&maps[0], BF16, q->data, 5, q_sizes, q_strides, q_box);
    const tq_dense_desc *kv[2] = {k, v};
    for (int i = 0; i < 2; ++i) {
        const int64_t sizes[3] = {tokens_kv, a.kv_heads, maps_batch}, strides[3] = {kv[i]->stride_t, kv[i]->stride_h, kv[i]->stride_b};
        ok = ok && encode(&maps[1 + i], BF16, kv[i]->data, 4, sizes, strides, kv_box);
    }
    if (!ok) {
        tq_set_cuda_error(cudaErrorInvalidValue, "tensor map of a prompt's queries, keys or values");
        return TQ_ERR_CUDA;
    }
    int device = 0;
    TQ_CUDA_CHECK(cudaGetDevice(&device));
    TQ_CUDA_CHECK(tq_allow_shared<tq_prompt_kernel<BF16>>(device, kSmem));
    const dim3 grid((unsigned)(a.batch * a.kv_heads * a.n_items), (unsigned)a.splits);
    tq_prompt_kernel<BF16><<<grid, kThreads, kSmem, stream>>>(maps[0], maps[1], maps[2], a);
    TQ_CUDA_CHECK(cudaGetLastError());
    if (a.splits > 1) {
        const int64_t rows = (int64_t)a.batch * a.n_q * a.kv_heads * a.group;
        tq_prompt_join_kernel<BF16><<<(unsigned)((rows + 3) / 4), 128, 0, stream>>>(a, rows);
        TQ_CUDA_CHECK(cudaGetLastError());
    }
    return TQ_OK;
}

int32_t prompt_attn(const tq_dense_desc *q, const tq_dense_desc *k, const tq_dense_desc *v, int32_t batch, int32_t q_heads,
                    int32_t kv_heads, int32_t n_q, int32_t n_kv, const int32_t *seq_start, const int32_t *cu_seqlens, int32_t total, float scale,
                    int32_t causal, void *workspace, size_t workspace_bytes, const tq_dense_desc *out, cudaStream_t stream) {
    if (!q || !k || !v || !out || !q->data || !k->data || !v->data || !out->data) return TQ_ERR_ARG;
    if (q->dtype != TQ_DTYPE_F16 && q->dtype != TQ_DTYPE_BF16) return q->dtype == TQ_DTYPE_F32 ? TQ_ERR_UNSUPPORTED : TQ_ERR_ARG;
    if (k->dtype != q->dtype || v->dtype != q->dtype || out->dtype != q->dtype) return TQ_ERR_ARG;
    if (batch < 0 || n_q < 0 || n_kv < 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads) return TQ_ERR_ARG;
    if (q_heads / kv_heads > TQ_MAX_PROMPT_GROUPS) return TQ_ERR_UNSUPPORTED;
    if (causal && n_kv < n_q) return TQ_ERR_ARG;
    const int64_t tokens_q = cu_seqlens ? total : n_q, tokens_kv = cu_seqlens ? total : n_kv;
    const int maps_batch = cu_seqlens ? 1 : batch;
    if (!aligned(q, maps_batch, q_heads, tokens_q) || !aligned(out, maps_batch, q_heads, tokens_q) || !aligned(k, maps_batch, kv_heads, tokens_kv) ||
        !aligned(v, maps_batch, kv_heads, tokens_kv))
        return TQ_ERR_ARG;
    if (((uintptr_t)seq_start | (uintptr_t)cu_seqlens) & 3 || (uintptr_t)workspace & 15) return TQ_ERR_ARG;
    const size_t need = tq_prompt_workspace_bytes(batch, q_heads, kv_heads, n_q, n_kv);
    if (workspace_bytes < need || (need && !workspace)) return TQ_ERR_WORKSPACE;
    if (batch == 0 || n_q == 0) return TQ_OK;
    if (n_kv == 0 || !(fabsf(scale) <= 3.4e38f)) return TQ_ERR_ARG;
    const Plan p = plan(batch, q_heads, kv_heads, n_q, n_kv);
    if ((int64_t)batch * kv_heads * p.n_items > 0x7fffffff) return TQ_ERR_UNSUPPORTED;
    PromptArgs a = {};
    a.out = const_cast<void *>(out->data), a.ob = out->stride_b, a.oh = out->stride_h, a.ot = out->stride_t;
    a.batch = batch, a.kv_heads = kv_heads, a.group = q_heads / kv_heads, a.positions = p.positions;
    a.n_q = n_q, a.n_kv = n_kv, a.total = total, a.n_items = p.n_items, a.tiles_per_cta = p.tiles_per_cta, a.splits = p.splits;
    a.seq_start = seq_start, a.cu_seqlens = cu_seqlens, a.causal = causal != 0, a.negate = scale < 0.f;
    a.scale_log2 = fmaxf(fabsf(scale) * 1.4426950408889634f, 1e-30f);  // (not 0: a masked logit is -inf and has to stay so)
    if (p.splits > 1) {
        const size_t rows = (size_t)batch * n_q * q_heads * p.splits;
        a.part_o = static_cast<float *>(workspace), a.part_ml = a.part_o + rows * TQ_D;
    }
    return q->dtype == TQ_DTYPE_BF16 ? launch<true>(q, k, v, tokens_q, tokens_kv, maps_batch, a, stream)
                                     : launch<false>(q, k, v, tokens_q, tokens_kv, maps_batch, a, stream);
}

}  // namespace

extern "C" size_t tq_prompt_workspace_bytes(int32_t batch, int32_t q_heads, int32_t kv_heads, int32_t n_q, int32_t n_kv) {
    if (batch <= 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || q_heads / kv_heads > kUmmaRows || n_q <= 0 || n_kv <= 0) return 0;
    const Plan p = plan(batch, q_heads, kv_heads, n_q, n_kv);
    return p.splits > 1 ? (size_t)batch * n_q * q_heads * p.splits * (TQ_D + 2) * sizeof(float) : 0;
}

extern "C" int32_t tq_prompt_attn(const tq_dense_desc *q, const tq_dense_desc *k, const tq_dense_desc *v, int32_t batch, int32_t q_heads,
                                  int32_t kv_heads, int32_t n_q, int32_t n_kv, const int32_t *seq_start, float scale, int32_t causal,
                                  void *workspace, size_t workspace_bytes, const tq_dense_desc *out, tq_stream stream) {
    TqRange range_("tq_prompt_attn");
    return prompt_attn(q, k, v, batch, q_heads, kv_heads, n_q, n_kv, seq_start, nullptr, 0, scale, causal, workspace, workspace_bytes, out,
                       (cudaStream_t)stream);
}

extern "C" int32_t tq_prompt_attn_packed(const tq_dense_desc *q, const tq_dense_desc *k, const tq_dense_desc *v, int32_t n_seqs,
                                         int32_t total, int32_t q_heads, int32_t kv_heads, const int32_t *cu_seqlens, int32_t max_seqlen,
                                         float scale, int32_t causal, void *workspace, size_t workspace_bytes, const tq_dense_desc *out,
                                         tq_stream stream) {
    TqRange range_("tq_prompt_attn_packed");
    if (!cu_seqlens || total < 0 || max_seqlen < 0 || (total == 0 && max_seqlen > 0 && n_seqs > 0)) return TQ_ERR_ARG;
    return prompt_attn(q, k, v, n_seqs, q_heads, kv_heads, max_seqlen, max_seqlen, nullptr, cu_seqlens, total, scale, causal, workspace,
                       workspace_bytes, out, (cudaStream_t)stream);
}

extern "C" int32_t tq_prompt_status(int32_t *status_out) {
    if (!status_out) return TQ_ERR_ARG;
    int v = 0;
    TQ_CUDA_CHECK(cudaDeviceSynchronize());  // (the copy alone does not wait for streams that do not block with the default one)
    TQ_CUDA_CHECK(cudaMemcpyFromSymbol(&v, g_prompt_status, sizeof(v)));
    *status_out = v;
    return TQ_OK;
}

extern "C" int32_t tq_prompt_status_clear(void) {
    const int v = 0;
    TQ_CUDA_CHECK(cudaMemcpyToSymbol(g_prompt_status, &v, sizeof(v)));
    return TQ_OK;
}
