// attention_prompt.cuh -- attention of chunks of new tokens over a paged cache
// on the tensor cores (tcgen05).
//
// The rows of a key head (tokens x the query heads that share it) are packed
// into tiles of 128; a CTA holds two such tiles, so that a block of 128 keys
// and values, once in shared memory, serves 256 rows.  For each block and tile
//   S = Q K^T        tcgen05.mma, Q and K in shared memory, S in tensor memory
//   P = exp2(S - m)  one thread a row: read S, running maximum m and sum, P as
//                    16-bit values into tensor memory
//   O += P V         tcgen05.mma, P in tensor memory, V in shared memory
// Roles: warps 0-3 and 4-7 the softmax of tile 0 and 1 (and its Q, and its
// result), warp 8 copies keys and values page by page (TMA boxes of as many
// rows as divide a page), warp 9 issues Q K^T and warp 10 P V.  P has a place of
// its own, so that the next S is computed while the softmax still works on this
// block; heads of 128 then leave room for a single S, which the tiles use in
// turn: a softmax moves it to registers at once, and the turns keep the tiles
// half a block apart, one in its softmax while the other has the tensor cores
// (left to themselves they fall into step).  A softmax thread rescales O in
// place, and only when the maximum has grown by more than 2^8, since any
// reference exponent in that range gives the same P / sum.
//
// A tile's keys end at its last row's position; only blocks that some row sees
// in part are masked.  In the first and last block V's rows outside the
// sequence are zeroed after the copy: their weights are zero, but what lies
// there may be NaN.
//
// With few tiles the blocks of a tile pair are split over several CTAs, whose
// parts (O, m, sum) attn_join_kernel adds up in order.
#pragma once

#include "attention.cuh"
#include "tcgen05.cuh"

namespace fmb {

constexpr uint32_t AP_THREADS = 384, AP_TILE = 128, AP_PAIR = 256, AP_KEYS = 128;
constexpr uint32_t AP_LEAST_BLOCKS = 4; // blocks a part of a split pair has at least

template <int DP> struct APrompt {
    static constexpr uint32_t HALVES = DP / 64;
    static constexpr uint32_t HALF = AP_KEYS * 128;        // 128 rows of 64 values
    static constexpr uint32_t BLOCK = HALVES * HALF;       // a Q tile, a K block, a V block
    static constexpr uint32_t STAGES = DP == 128 ? 5 : 8;
    // Tensor memory, 512 columns: P (64) and O (DP) of each tile, and S (128): one of each
    // tile where there is room, else one that the tiles use in turn.
    static constexpr bool ONE_S = DP == 128;
    __host__ __device__ static constexpr uint32_t o_col(uint32_t t) { return t * DP; }
    __host__ __device__ static constexpr uint32_t p_col(uint32_t t) { return 2 * DP + t * 64; }
    __host__ __device__ static constexpr uint32_t s_col(uint32_t t) { return 2 * DP + 128 + (ONE_S ? 0 : t * 128); }
    static constexpr uint32_t OFF_KV = 2 * BLOCK;
    static constexpr uint32_t OFF_BAR = OFF_KV + STAGES * BLOCK;
    static constexpr uint32_t SMEM = OFF_BAR + 512 + 1024; // and the alignment to 1024
};

struct APParams {
    AttnParams a;
    uint32_t box_rows; // rows of a TMA box: the largest power of two that divides a page, at most 128
    bool heads_first;  // the tensor maps' second dimension is the heads, not a page's rows
    uint32_t splits;
    float *part;       // [pair][head][split][256][DP]
    float2 *part_ml;
};

// ---- descriptors ----------------------------------------------------------------

template <bool BF16> __device__ constexpr uint32_t ap_idesc(uint32_t n, bool b_rows_are_k) {
    return (1u << 4) | ((BF16 ? 1u : 0u) << 7) | ((BF16 ? 1u : 0u) << 10) | ((b_rows_are_k ? 1u : 0u) << 16) |
           ((n >> 3) << 17) | ((128u >> 4) << 24);
}

// V as the B operand: rows are keys (the K dimension), 64 values of N contiguous in
// 128-byte swizzled rows; the next 64 values lie a half further, the next 8 keys 1024 bytes.
__device__ __forceinline__ uint64_t ap_desc_v(uint32_t saddr, uint32_t half_bytes) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((saddr >> 4) & 0x3FFFu);
    d |= static_cast<uint64_t>(half_bytes >> 4) << 16;
    d |= static_cast<uint64_t>(1024u >> 4) << 32;
    d |= static_cast<uint64_t>(1u) << 46;
    d |= static_cast<uint64_t>(2u) << 61;
    return d;
}

// D[tmem] (+)= A[smem] x B[smem]^T, issued by one thread.
__device__ __forceinline__ void mma_f16_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                 " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
                 "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
                 : "memory");
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, int32_t x, int32_t y, int32_t z,
                                            int32_t page, uint64_t *bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, "
                 "%4, %5}], [%6];\n" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(page), "r"(smem_u32(bar))
                 : "memory");
}

__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }

// Uses of v stay behind this point (a wait for tensor-memory loads does not name their registers).
template <int N> __device__ __forceinline__ void pin(uint32_t (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 8)
        asm volatile("" : "+r"(v[i]), "+r"(v[i + 1]), "+r"(v[i + 2]), "+r"(v[i + 3]), "+r"(v[i + 4]), "+r"(v[i + 5]),
                          "+r"(v[i + 6]), "+r"(v[i + 7]));
}

__device__ __forceinline__ uint64_t pack_f32x2(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpack_f32x2(uint64_t v, float &lo, float &hi) {
    asm("mov.b64 {%0, %1}, %2;\n" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;\n" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Bounded wait that also gives up once another role has.
__device__ __forceinline__ bool ap_wait(uint64_t *bar, uint32_t parity, volatile uint32_t *abort_flag, int *status) {
    if (mbar_try_wait(bar, parity)) return true;
    const long long start = clock64();
    for (uint32_t it = 1;; ++it) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((it & 63u) == 0) {
            if (*abort_flag) return false;
            if (clock64() - start > (1ll << 31)) {
                *abort_flag = 1;
                raise_device_status(status, FM_STATUS_INTERNAL_ERROR);
                return false;
            }
        }
    }
}

// ---- shape of a pair of tiles -----------------------------------------------------

__device__ __forceinline__ uint32_t ap_pairs(const AttnParams &p, const AttnSeq &s) {
    const uint64_t rows = static_cast<uint64_t>(s.ql) * p.group;
    return rows > p.row_limit ? static_cast<uint32_t>((rows + AP_PAIR - 1) / AP_PAIR) : 0;
}

// Keys [lo, hi) seen by rows [row0, row0 + 128) of the sequence, blocks [j0, j1), and the
// blocks that every row of the tile sees whole: those inside [whole_lo, whole_hi).
struct APTile {
    uint32_t rows, j0, j1;
    uint32_t whole_lo, whole_hi;
};
__device__ __forceinline__ APTile ap_tile(const AttnParams &p, const AttnSeq &s, uint32_t row0) {
    APTile t{};
    const uint64_t all = static_cast<uint64_t>(s.ql) * p.group;
    if (row0 >= all) return t;
    t.rows = all - row0 < AP_TILE ? static_cast<uint32_t>(all - row0) : AP_TILE;
    const int64_t base = static_cast<int64_t>(s.kl) - s.ql;
    const int64_t first = base + row0 / p.group, last = base + (row0 + t.rows - 1) / p.group;
    const int64_t hi = p.causal ? last + 1 : s.kl;
    int64_t lo = p.window ? first - p.window + 1 : 0;
    if (lo < 0) lo = 0;
    const int64_t whole_hi = p.causal ? first + 1 : s.kl, whole_lo = p.window ? last - p.window + 1 : 0;
    t.whole_hi = whole_hi > 0 ? static_cast<uint32_t>(whole_hi) : 0;
    t.whole_lo = whole_lo > 0 ? static_cast<uint32_t>(whole_lo) : 0;
    if (hi > lo) {
        t.j0 = static_cast<uint32_t>(lo / AP_KEYS);
        t.j1 = static_cast<uint32_t>((hi + AP_KEYS - 1) / AP_KEYS);
    }
    return t;
}

// Row r of tile t of a pair: its token and query head.
struct APRow {
    uint64_t token, qhead;
    bool valid;
};
__device__ __forceinline__ APRow ap_row(const AttnParams &p, const AttnSeq &s, uint32_t head, uint32_t pair, uint32_t t,
                                        uint32_t r) {
    const uint32_t row = pair * AP_PAIR + t * AP_TILE + r, tok = row / p.group;
    return {static_cast<uint64_t>(s.q0) + tok, static_cast<uint64_t>(head) * p.group + (row - tok * p.group), tok < s.ql};
}

// The blocks of a pair, and how many parts they are split into.
struct APSpan {
    uint32_t j0, j1, parts;
};
__device__ __forceinline__ APSpan ap_span(const APTile &t0, const APTile &t1, uint32_t splits) {
    APSpan r;
    const bool e0 = t0.j1 > t0.j0, e1 = t1.j1 > t1.j0;
    r.j0 = e0 ? t0.j0 : e1 ? t1.j0 : 0;
    r.j1 = e1 ? (e0 && t0.j1 > t1.j1 ? t0.j1 : t1.j1) : e0 ? t0.j1 : 0;
    const uint32_t n = (r.j1 - r.j0) / AP_LEAST_BLOCKS;
    r.parts = n < 1 ? 1 : n < splits ? n : splits;
    return r;
}
__device__ __forceinline__ uint32_t ap_part_begin(const APSpan &s, uint32_t part) {
    return s.j0 + static_cast<uint32_t>(static_cast<uint64_t>(s.j1 - s.j0) * part / s.parts);
}

// ---- the kernel ---------------------------------------------------------------------

template <int DP, bool BF16>
__global__ void __launch_bounds__(AP_THREADS, 1)
    attn_prompt_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                       const __grid_constant__ APParams pp) {
    using L = APrompt<DP>;
    const AttnParams &p = pp.a;
    extern __shared__ uint8_t ap_smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(ap_smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::OFF_BAR);
    uint64_t *q_full = bars, *s_full = bars + 2, *p_full = bars + 4, *o_done = bars + 6, *edge = bars + 8;
    uint64_t *s_free = bars + 9, *drain = bars + 11, *kv_full = bars + 13, *kv_empty = kv_full + L::STAGES;
    // TMEM base, abort, the pair's sequence, the pair in it and among all
    uint32_t *misc = reinterpret_cast<uint32_t *>(kv_empty + L::STAGES);
    volatile uint32_t *abort_flag = misc + 1;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;

    // ---- which pair of which sequence ------------------------------------------------
    const uint32_t head = blockIdx.x % p.kv_heads;
    const uint32_t part = blockIdx.x / p.kv_heads % pp.splits;
    const uint32_t rank = blockIdx.x / p.kv_heads / pp.splits;
    if (warp == 0) {
        // the longest tiles of a sequence are its last: pairs are taken from the end
        uint32_t total = 0;
        for (uint32_t b0 = 0; b0 < p.seqs; b0 += 32) {
            const uint32_t n = b0 + lane < p.seqs ? ap_pairs(p, attn_seq(p, b0 + lane, blockIdx.x == 0)) : 0;
            total += __reduce_add_sync(0xFFFFFFFFu, n);
        }
        if (lane == 0) misc[2] = 0xFFFFFFFFu;
        __syncwarp();
        if (rank < total) {
            const uint32_t want = total - 1 - rank;
            uint32_t before = 0;
            for (uint32_t b0 = 0; b0 < p.seqs && before <= want; b0 += 32) {
                const uint32_t n = b0 + lane < p.seqs ? ap_pairs(p, attn_seq(p, b0 + lane, false)) : 0;
                uint32_t inc = n;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t t = __shfl_up_sync(0xFFFFFFFFu, inc, o);
                    if (lane >= static_cast<uint32_t>(o)) inc += t;
                }
                const uint32_t at = before + inc - n;
                if (n && want >= at && want < at + n) {
                    misc[2] = b0 + lane;
                    misc[3] = want - at;
                    misc[4] = want;
                }
                before += __shfl_sync(0xFFFFFFFFu, inc, 31);
            }
        }
    } else if (threadIdx.x == 32) {
        for (uint32_t i = 0; i < 2; ++i) {
            mbar_init(&q_full[i], 128);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 128);
            mbar_init(&o_done[i], 1);
            mbar_init(&s_free[i], 128);
            mbar_init(&drain[i], 1);
        }
        mbar_init(edge, 1);
        for (uint32_t i = 0; i < L::STAGES; ++i) {
            mbar_init(&kv_full[i], 1);
            mbar_init(&kv_empty[i], 1);
        }
        misc[1] = 0;
        fence_barrier_init();
    }
    __syncthreads();
    const uint32_t b = misc[2], pair = misc[3];
    if (b == 0xFFFFFFFFu) return;
    const AttnSeq s = attn_seq(p, b, false);
    const APTile tile0 = ap_tile(p, s, pair * AP_PAIR), tile1 = ap_tile(p, s, pair * AP_PAIR + AP_TILE);
    const APSpan span = ap_span(tile0, tile1, pp.splits);
    if (part >= span.parts) return;
    const uint32_t jb = ap_part_begin(span, part), je = ap_part_begin(span, part + 1);

    if (warp == 11) {
        tmem_alloc(misc, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = misc[0];

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;\n");
        if (warp == 8) {
            // ---- keys and values ----------------------------------------------------
            const uint32_t R = pp.box_rows, n_boxes = AP_KEYS / R;
            uint32_t it = 0, edges = 0;
            bool going = true;
            for (uint32_t j = jb; j < je && going; ++j) {
                const uint32_t key = j * AP_KEYS + lane * R;
                const bool live = lane < n_boxes && key < s.kl && key + R > s.lo;
                int32_t page = 0, row = 0;
                if (live) {
                    const uint32_t at = key / p.page_size;
                    row = static_cast<int32_t>(key - at * p.page_size);
                    page = __ldg(p.table + b * p.tb + at);
                    if (page < 0 || static_cast<uint32_t>(page) >= p.n_pages) {
                        raise_device_status(p.status, FM_STATUS_INVALID_ARGUMENT);
                        page = -1; // outside the tensor map: the box is filled with zeros
                    }
                }
                const uint32_t bytes = __popc(__ballot_sync(0xFFFFFFFFu, live)) * R * 128 * L::HALVES;
                const bool at_edge = j * AP_KEYS < s.lo || (j + 1) * AP_KEYS > s.kl;
#pragma unroll
                for (uint32_t kind = 0; kind < 2; ++kind, ++it) {
                    const uint32_t st = it % L::STAGES;
                    if (!ap_wait(&kv_empty[st], ((it / L::STAGES) & 1u) ^ 1u, abort_flag, p.status)) {
                        going = false;
                        break;
                    }
                    const uint32_t dst = smem_u32(smem + L::OFF_KV + st * L::BLOCK);
                    uint64_t *bar = kind == 1 && at_edge ? edge : &kv_full[st];
                    if (lane == 0) mbar_expect_tx(bar, bytes);
                    __syncwarp();
                    if (live) {
#pragma unroll
                        for (uint32_t h = 0; h < L::HALVES; ++h)
                            tma_load_4d(dst + h * L::HALF + lane * R * 128, kind ? &map_v : &map_k,
                                        static_cast<int32_t>(h * 64), pp.heads_first ? static_cast<int32_t>(head) : row,
                                        pp.heads_first ? row : static_cast<int32_t>(head), page, bar);
                    }
                    if (kind == 1 && at_edge) {
                        if (!ap_wait(edge, edges & 1u, abort_flag, p.status)) {
                            going = false;
                            break;
                        }
                        ++edges;
                        for (uint32_t r = lane; r < AP_KEYS; r += 32) {
                            const uint32_t k = j * AP_KEYS + r;
                            if (k >= s.lo && k < s.kl) continue;
#pragma unroll
                            for (uint32_t x = 0; x < L::HALVES * 8; ++x)
                                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};\n" ::"r"(
                                                 dst + (x >> 3) * L::HALF + r * 128 + (x & 7u) * 16),
                                             "r"(0)
                                             : "memory");
                        }
                        fence_proxy_async();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&kv_full[st]);
                    }
                }
            }
            // what was asked for must land before the CTA's shared memory goes away
            if (!going)
                for (uint32_t i = it > L::STAGES ? it - L::STAGES : 0; i < it; ++i)
                    (void)mbar_wait(&kv_full[i % L::STAGES], (i / L::STAGES) & 1u);
        } else if ((warp == 9 || warp == 10) && lane == 0) {
            // ---- the products: warp 9 S = Q K^T, warp 10 O += P V -----------------------
            // S is asked for as soon as its place is free, so that it waits for its softmax
            // and not the other way round; the tensor cores take what is ready.
            const bool scores = warp == 9;
            constexpr uint32_t id_s = ap_idesc<BF16>(AP_KEYS, false), id_o = ap_idesc<BF16>(DP, true);
            uint32_t it = scores ? 0 : 1; // load of block jb's keys, or values
            uint32_t n0 = 0, n1 = 0, s_used = 0;
            bool ok = true;
            for (uint32_t j = jb; j < je && ok; ++j, it += 2) {
                const uint32_t st = it % L::STAGES;
                const uint32_t kv = smem_u32(smem + L::OFF_KV + st * L::BLOCK);
                ok = ap_wait(&kv_full[st], (it / L::STAGES) & 1u, abort_flag, p.status);
#pragma unroll
                for (uint32_t t = 0; t < 2; ++t) {
                    const APTile &tile = t ? tile1 : tile0;
                    uint32_t &n = t ? n1 : n0;
                    if (!ok || j < tile.j0 || j >= tile.j1) continue;
                    if (scores) {
                        if (n == 0) ok = ap_wait(&q_full[t], 0, abort_flag, p.status);
                        const uint32_t used = L::ONE_S ? s_used : n;
                        if (ok && used) ok = ap_wait(&s_free[L::ONE_S ? 0 : t], (used - 1) & 1u, abort_flag, p.status);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t q_addr = smem_u32(smem + t * L::BLOCK);
#pragma unroll
                        for (uint32_t k = 0; k < DP / 16; ++k) {
                            const uint32_t off = (k >> 2) * L::HALF + (k & 3u) * 32;
                            mma_f16_ss(tmem + L::s_col(t), smem_desc_sw128(q_addr + off), smem_desc_sw128(kv + off),
                                       id_s, k != 0);
                        }
                        tc_commit(&s_full[t]);
                        ++s_used;
                    } else {
                        ok = ap_wait(&p_full[t], n & 1u, abort_flag, p.status);
                        if (!ok) break;
                        tc_fence_after();
#pragma unroll
                        for (uint32_t k = 0; k < AP_KEYS / 16; ++k)
                            mma_f16_ts(tmem + L::o_col(t), tmem + L::p_col(t) + k * 8,
                                       ap_desc_v(kv + k * 2048, L::HALF), id_o, (n | k) != 0);
                        tc_commit(&o_done[t]);
                    }
                    ++n;
                }
                if (ok) tc_commit(&kv_empty[st]);
            }
            // every product and commit must have ended before tensor and shared memory go away
            tc_commit(&drain[scores ? 0 : 1]);
            (void)mbar_wait(&drain[scores ? 0 : 1], 0);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;\n");
        // ---- softmax: one thread a row ------------------------------------------------
        const uint32_t t = warp >> 2, r = threadIdx.x & 127u;
        const APTile tile = t ? tile1 : tile0;
        const uint32_t lane_addr = ((warp & 3u) * 32u) << 16;
        const uint32_t s_tmem = tmem + (t ? L::s_col(1) : L::s_col(0)) + lane_addr;
        const uint32_t p_tmem = tmem + (t ? L::p_col(1) : L::p_col(0)) + lane_addr;
        const uint32_t o_tmem = tmem + (t ? L::o_col(1) : L::o_col(0)) + lane_addr;
        // Q, rows past the end as zeros
        {
            const APRow w = ap_row(p, s, head, pair, t, r);
            const uint16_t *src = static_cast<const uint16_t *>(p.q) + w.token * p.qt + w.qhead * p.qh;
            const uint32_t dst = smem_u32(smem + t * L::BLOCK) + r * 128;
#pragma unroll
            for (uint32_t c = 0; c < DP / 8; ++c) {
                uint4 v = make_uint4(0, 0, 0, 0);
                if (w.valid && c * 8 < p.dim) v = *reinterpret_cast<const uint4 *>(src + c * 8);
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(dst + (c >> 3) * L::HALF +
                                                                              (((c & 7u) ^ (r & 7u)) << 4)),
                             "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
                             : "memory");
            }
            fence_proxy_async();
            mbar_arrive(&q_full[t]);
        }
        uint32_t key_lo = 0, key_hi = s.kl;
        if (r < tile.rows) {
            const int64_t pos = static_cast<int64_t>(s.kl) - s.ql + (pair * AP_PAIR + t * AP_TILE + r) / p.group;
            const int64_t hi = p.causal ? pos + 1 : s.kl, lo = p.window ? pos - p.window + 1 : 0;
            key_hi = hi > 0 ? static_cast<uint32_t>(hi) : 0;
            key_lo = lo > 0 ? static_cast<uint32_t>(lo) : 0;
        }
        const uint32_t tb = tile.j0 > jb ? tile.j0 : jb, te = tile.j1 < je ? tile.j1 : je;
        const uint32_t blocks = te > tb ? te - tb : 0;
        float m = -INFINITY; // in log2
        uint64_t sum2 = 0;   // two f32 sums
        const uint64_t scale2 = pack_f32x2(p.scale_log2, p.scale_log2);
        bool ok = true;
        for (uint32_t n = 0; n < blocks; ++n) {
            ok = ap_wait(&s_full[t], n & 1u, abort_flag, p.status);
            if (!ok) break;
            tc_fence_after();
            uint32_t x[4][32];
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_ld32(s_tmem + c * 32, x[c]);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 4; ++c) pin(x[c]);
            tc_fence_before();
            mbar_arrive(&s_free[L::ONE_S ? 0 : t]);
            const uint32_t key0 = (tb + n) * AP_KEYS;
            if (key0 + AP_KEYS > tile.whole_hi || key0 < tile.whole_lo) {
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const uint32_t key = key0 + c * 32 + i;
                        if (key < key_lo || key >= key_hi) x[c][i] = 0xFF800000u; // -inf
                    }
            }
            float top[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                top[c] = __uint_as_float(x[c][0]);
#pragma unroll
                for (int i = 1; i < 31; i += 2)
                    top[c] = max3(top[c], __uint_as_float(x[c][i]), __uint_as_float(x[c][i + 1]));
                top[c] = fmaxf(top[c], __uint_as_float(x[c][31]));
            }
            const float high = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * p.scale_log2;
            if (__any_sync(0xFFFFFFFFu, high > m + 8.0f)) {
                const float to = fmaxf(m, high);
                const float f = m == -INFINITY ? 0.0f : exp2_approx(m - to);
                m = to;
                if (n) { // the last block's product has written O
                    ok = ap_wait(&o_done[t], (n - 1) & 1u, abort_flag, p.status);
                    if (!ok) break;
                    tc_fence_after();
                    float a, c2;
                    unpack_f32x2(sum2, a, c2);
                    sum2 = pack_f32x2(a * f, c2 * f);
#pragma unroll
                    for (int c = 0; c < DP / 16; ++c) {
                        uint32_t o[16];
                        tmem_ld16(o_tmem + c * 16, o);
                        tmem_wait_ld();
                        pin(o);
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                        tmem_st16(o_tmem + c * 16, o);
                    }
                }
            }
            const float base = m == -INFINITY ? 0.0f : -m;
            const uint64_t base2 = pack_f32x2(base, base);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t w[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float a, c2;
                    unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(x[c][2 * i]), __uint_as_float(x[c][2 * i + 1])),
                                           scale2, base2),
                                 a, c2);
                    a = exp2_approx(a);
                    c2 = exp2_approx(c2);
                    sum2 = add_f32x2(sum2, pack_f32x2(a, c2));
                    w[i] = pack_pair<BF16>(a, c2);
                }
                if (c == 0 && n) { // the last block's product has read P
                    ok = ap_wait(&o_done[t], (n - 1) & 1u, abort_flag, p.status);
                    if (!ok) break;
                    tc_fence_after();
                }
                tmem_st16(p_tmem + c * 16, w);
            }
            if (!ok) break;
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&p_full[t]);
        }
        // ---- result -------------------------------------------------------------------
        if (ok && blocks) ok = ap_wait(&o_done[t], (blocks - 1) & 1u, abort_flag, p.status);
        if (ok && tile.rows) {
            tc_fence_after();
            float a, c2;
            unpack_f32x2(sum2, a, c2);
            const float sum = blocks ? a + c2 : 0.0f;
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            // where the row goes is worked out again: kept over the loop it would cost registers
            uint32_t again = r;
            asm volatile("" : "+r"(again));
            const AttnSeq s2 = attn_seq(p, misc[2], false);
            const APRow w = ap_row(p, s2, head, misc[3], t, again);
            uint16_t *out = static_cast<uint16_t *>(p.out) + w.token * p.ot + w.qhead * p.oh;
            const uint64_t slot =
                ((static_cast<uint64_t>(misc[4]) * p.kv_heads + head) * pp.splits + part) * AP_PAIR + t * AP_TILE + r;
#pragma unroll
            for (int c = 0; c < DP / 32; ++c) {
                uint32_t o[32];
                if (blocks) {
                    tmem_ld32(o_tmem + c * 32, o);
                    tmem_wait_ld();
                    pin(o);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = 0;
                }
                if (!w.valid) continue;
                if (span.parts == 1) {
                    uint16_t *dst = out + c * 32;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t v[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            v[k] = pack_pair<BF16>(__uint_as_float(o[i * 8 + 2 * k]) * inv,
                                                   __uint_as_float(o[i * 8 + 2 * k + 1]) * inv);
                        if (c * 32u + i * 8u < p.dim)
                            *reinterpret_cast<uint4 *>(dst + i * 8) = make_uint4(v[0], v[1], v[2], v[3]);
                    }
                } else {
                    uint4 *dst = reinterpret_cast<uint4 *>(pp.part + slot * DP + c * 32);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        dst[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                }
            }
            if (w.valid) {
                if (span.parts > 1)
                    pp.part_ml[slot] = make_float2(m, sum);
                else if (p.lse)
                    p.lse[w.token * p.heads + w.qhead] =
                        sum == 0.0f ? -INFINITY : m * 0.6931471805599453f + logf(sum);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 11) tmem_dealloc(tmem, 512);
}

// Adds up the parts of split pairs: a warp a row.
template <int DP, bool BF16> __global__ void __launch_bounds__(256) attn_join_kernel(const __grid_constant__ APParams pp) {
    constexpr int V = DP / 32;
    const AttnParams &p = pp.a;
    const uint32_t lane = threadIdx.x & 31u;
    const uint64_t id = static_cast<uint64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    const uint64_t qhead = id % p.heads;
    const uint32_t t = static_cast<uint32_t>(id / p.heads);
    if (t >= p.tokens) return;
    // the token's sequence, and the pairs before it
    uint32_t before = 0, b = 0;
    bool found = false;
    AttnSeq s{};
    for (uint32_t b0 = 0; b0 < p.seqs && !found; b0 += 32) {
        AttnSeq mine{};
        if (b0 + lane < p.seqs) mine = attn_seq(p, b0 + lane, false);
        const uint32_t n = ap_pairs(p, mine);
        const uint32_t hit = __ballot_sync(0xFFFFFFFFu, n && t >= mine.q0 && t < mine.q0 + mine.ql);
        const uint32_t at = hit ? __ffs(hit) - 1 : 32;
        before += __reduce_add_sync(0xFFFFFFFFu, lane < at ? n : 0u);
        if (hit) {
            found = true;
            b = b0 + at;
        }
    }
    if (!found) return;
    s = attn_seq(p, b, false);
    const uint32_t head = static_cast<uint32_t>(qhead) / p.group, g = static_cast<uint32_t>(qhead) % p.group;
    const uint32_t row = (t - s.q0) * p.group + g, pair = row / AP_PAIR;
    const APSpan span =
        ap_span(ap_tile(p, s, pair * AP_PAIR), ap_tile(p, s, pair * AP_PAIR + AP_TILE), pp.splits);
    if (span.parts == 1) return; // written by its one CTA
    const uint64_t slot0 =
        ((static_cast<uint64_t>(before + pair) * p.kv_heads + head) * pp.splits) * AP_PAIR + row % AP_PAIR;
    float top = -INFINITY;
    for (uint32_t i = 0; i < span.parts; ++i) top = fmaxf(top, pp.part_ml[slot0 + i * AP_PAIR].x);
    float acc[V] = {}, sum = 0.0f;
    for (uint32_t i = 0; i < span.parts; ++i) {
        const uint64_t slot = slot0 + static_cast<uint64_t>(i) * AP_PAIR;
        const float2 ml = pp.part_ml[slot];
        const float f = ml.x == -INFINITY ? 0.0f : exp2_approx(ml.x - top);
        sum += ml.y * f;
#pragma unroll
        for (int x = 0; x < V; ++x) acc[x] += pp.part[slot * DP + lane * V + x] * f;
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    uint16_t *dst = static_cast<uint16_t *>(p.out) + t * p.ot + qhead * p.oh;
#pragma unroll
    for (int x = 0; x < V; x += 2)
        if (lane * V + x < p.dim)
            *reinterpret_cast<uint32_t *>(dst + lane * V + x) = pack_pair<BF16>(acc[x] * inv, acc[x + 1] * inv);
    if (p.lse && lane == 0)
        p.lse[static_cast<uint64_t>(t) * p.heads + qhead] =
            sum == 0.0f ? -INFINITY : top * 0.6931471805599453f + logf(sum);
}

} // namespace fmb
