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
// Roles: warps 0-3 and 4-7 the softmax of tile 0 and 1 and its result; warp 8
// walks through the CTA's work, tells the others of each segment, and copies its
// keys and values page by page (TMA boxes of as many rows as divide a page);
// warp 9 issues Q K^T and warp 10 P V; warp 11 copies Q.  P has a place of its
// own, so that the next S is computed while the softmax still works on this
// block.  There is one S, which the tiles use in turn: a softmax moves it to
// registers at once, and the turns keep the tiles apart, one in its exponentials
// while the other waits (left to themselves they fall into step).  Heads of 64
// have room for an S each, but that was 5% slower.  With heads of 128 there is
// none beside a P with columns of its own; with P over S's columns two S fit, as
// in an early form of this kernel, which took 617 us where P's own columns then
// took 492 (a prompt of 8192; not tried again with the later steps around it).
// A softmax thread rescales O in place, and only when the maximum has
// grown by more than 2^8, since any reference exponent in that range gives the
// same P / sum.
//
// P is rounded to the cache's 16-bit type because the matrix instructions take
// both operands in one type; the sums take it unrounded.  For bf16 the result is then
// within 0.0021 to 0.0023 of the 64-bit form (relative, as a norm), of which its own
// rounding is 0.0017.
//
// A tile's keys end at its last row's position; only blocks that some row sees
// in part are masked.  In the first and last block V's rows outside the
// sequence are zeroed after the copy: their weights are zero, but what lies
// there may be NaN.
//
// A persistent CTA an SM.  Where there are many (pair of tiles, key head) items,
// they go to the CTAs whole, the longest first, in rounds that run there and
// back.  Where there are few, all their blocks laid end to end are cut into equal
// ranges, one a CTA; the cut items' fragments (O, m, sum) are added up in order
// by attn_join_kernel.  A CTA has at most two: of the item that began before its
// range and of the one that goes on after it.  Where there are fewer items than CTAs,
// each is cut into pieces of its own, so that no CTA begins a second item (8 chunks of 128
// behind 2000 keys: 69 -> 51 us).
//
// Measured: a prompt of 8192, 32/8 heads of 128, bf16: 505 to 550 us by machine and heat, 1.0
// to 1.1 PFLOP/s of the 1.66 of a library product, with the tensor pipe 54% busy and the
// exponentials 54% at 1.64 GHz (the power cap): a block's two tiles take 3200 cycles where
// either alone would take 2048.  Chunks behind contexts, heads of 64: 160 us; the exponentials
// alone are 80 of them, the special-function unit is 58% busy.
#pragma once

#include "attention_rows.cuh"

namespace fmb {

constexpr uint32_t AP_THREADS = 384, AP_TILE = 128, AP_PAIR = 256, AP_KEYS = 128;
// Where blocks are dealt out: what an item costs beside its blocks (its Q, its
// result), in blocks, and the least that a CTA takes.  Where each CTA has a piece of
// one item: its least blocks, and the blocks that cutting the longest item has to
// save, for the fragments and their join.
constexpr uint32_t AP_ITEM_COST = 5, AP_LEAST_COST = 6 + AP_ITEM_COST;
constexpr uint32_t AP_LEAST_PIECE = 4, AP_LEAST_SAVED = 4;
constexpr uint32_t AP_MAX_PAIRS = 1024; // pairs of tiles whose blocks can be dealt out

template <int DP> struct APrompt {
    static constexpr uint32_t HALVES = DP / 64;
    static constexpr uint32_t HALF = AP_KEYS * 128;        // 128 rows of 64 values
    static constexpr uint32_t BLOCK = HALVES * HALF;       // a Q tile, a K block, a V block
    static constexpr uint32_t STAGES = DP == 128 ? 5 : 8;
    // Tensor memory, 512 columns: O (DP) and P (64) of each tile, and one S (128).
    __host__ __device__ static constexpr uint32_t o_col(uint32_t t) { return t * DP; }
    __host__ __device__ static constexpr uint32_t p_col(uint32_t t) { return 2 * DP + t * 64; }
    static constexpr uint32_t S_COL = 2 * DP + 128;
    static constexpr uint32_t OFF_KV = 2 * BLOCK;
    static constexpr uint32_t OFF_BAR = OFF_KV + STAGES * BLOCK;
    static constexpr uint32_t OFF_SEG = OFF_BAR + 512;
    static constexpr uint32_t SMEM = OFF_SEG + 512 + 1024; // and the alignment to 1024
};

struct APParams {
    AttnParams a;
    uint32_t box_rows; // rows of a TMA box: the largest power of two that divides a page, at most 128
    bool heads_first;  // the tensor maps' second dimension is the heads, not a page's rows
    bool wide;         // rows of out lie and end on 32 bytes
    bool deal;         // blocks are dealt out, not items
    uint32_t max_pairs;
    uint32_t ctas;     // CTAs of the prompt kernel; the others of attn_beside_kernel take few-row sequences
    ARForm rows_form;  // and how: a CTA a unit, a warp a unit, or even ranges
    uint32_t rows_tiles, rows_warps; // row tiles a unit's sequence and head; warps that a unit each takes
    float *part;       // [CTA][began before, goes on][256][DP]
    float2 *part_ml;
    int4 *tail;        // [CTA] the item that goes on after it: sequence (or -1), pair, head, fragments
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

// A 32-byte store: a thread holds a whole row, and anything shorter would leave sectors
// half written.
__device__ __forceinline__ void store_32b(void *dst, const uint32_t *v) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"l"(dst), "r"(v[0]), "r"(v[1]),
                 "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

// Largest of three or two; NaN if one is.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;\n" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float max2(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Bounded wait of a whole warp that also gives up once another role has; the
// same answer in every lane.  (All lanes poll: with one, and the others waiting
// for it, a prompt of 8192 tokens took 730 us where it then took 460, single calls on a
// cool GPU.)
__device__ __forceinline__ bool ap_wait(uint64_t *bar, uint32_t parity, volatile uint32_t *abort_flag, int *status) {
    bool done = mbar_try_wait(bar, parity);
    if (!done) {
        const long long start = clock64();
        for (uint32_t it = 1;; ++it) {
            done = mbar_try_wait(bar, parity);
            if (done) break;
            if ((it & 63u) == 0) {
                if (*abort_flag) break;
                if (clock64() - start > (1ll << 31)) {
                    *abort_flag = 1;
                    raise_device_status(status, FM_STATUS_INTERNAL_ERROR);
                    break;
                }
            }
        }
    }
    return __all_sync(0xFFFFFFFFu, done);
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

// The blocks of a pair; one without keys has a block that no tile takes.
__device__ __forceinline__ uint2 ap_span(const APTile &t0, const APTile &t1) {
    const bool e0 = t0.j1 > t0.j0, e1 = t1.j1 > t1.j0;
    const uint32_t j0 = e0 ? t0.j0 : e1 ? t1.j0 : 0;
    const uint32_t j1 = e1 ? (e0 && t0.j1 > t1.j1 ? t0.j1 : t1.j1) : e0 ? t0.j1 : 0;
    return make_uint2(j0, j1 > j0 ? j1 : j0 + 1);
}

// A CTA's way through its work, walked by each role for itself.
struct APWalk {
    uint32_t b, pair, head, off; // dealt blocks: the next item, and the cost of it that is not this CTA's
    uint64_t left;               // cost left; or items in all
    uint32_t round;              // dealt items
    uint32_t piece;              // blocks of a piece where each CTA has one piece of one item; else 0
};
struct APSeg {
    AttnSeq s;
    APTile t0, t1;
    uint32_t b, pair, head, jb, je, j1; // blocks [jb, je); the item's end
    bool starts, whole;
};

// What the other roles have to know of a segment, in shared memory.
constexpr uint32_t AP_SEG_SLOTS = 4, AP_SEG_READERS = 11; // eight softmax warps, two issuers, Q
struct APShared {
    uint32_t jb, je;                     // je == 0: the end
    uint32_t tb[2], te[2];               // the blocks of each tile among them
    uint32_t whole_lo[2], whole_hi[2];
    uint32_t rows[2];
    uint32_t row0;                       // first row of the pair
    uint32_t q0, ql, kl, head;
    uint32_t starts, whole;
};
static_assert(sizeof(APShared) * AP_SEG_SLOTS <= 512, "segments outgrow their place");

// Called by whole warps; false at the end.
__device__ __forceinline__ bool ap_next(const APParams &pp, APWalk &w, APSeg &g) {
    const AttnParams &p = pp.a;
    const uint32_t lane = threadIdx.x & 31u;
    if (!pp.deal) {
        const uint64_t rank = static_cast<uint64_t>(w.round) * pp.ctas +
                              (w.round & 1u ? pp.ctas - 1 - blockIdx.x : blockIdx.x);
        if (rank >= w.left) return false;
        ++w.round;
        const uint64_t item = w.left - 1 - rank; // the longest tiles of a sequence are its last
        const uint32_t want = static_cast<uint32_t>(item / p.kv_heads);
        w.head = static_cast<uint32_t>(item - static_cast<uint64_t>(want) * p.kv_heads);
        uint32_t before = 0;
        w.b = 0;
        for (uint32_t b0 = 0; b0 < p.seqs; b0 += 32) {
            const uint32_t n = b0 + lane < p.seqs ? ap_pairs(p, attn_seq(p, b0 + lane, false)) : 0;
            uint32_t inc = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t t = __shfl_up_sync(0xFFFFFFFFu, inc, o);
                if (lane >= static_cast<uint32_t>(o)) inc += t;
            }
            const uint32_t hit = __ballot_sync(0xFFFFFFFFu, want < before + inc);
            if (hit) {
                const uint32_t at = __ffs(hit) - 1;
                w.b = b0 + at;
                w.pair = want - before - __shfl_sync(0xFFFFFFFFu, inc - n, at);
                break;
            }
            before += __shfl_sync(0xFFFFFFFFu, inc, 31);
        }
    }
    do {
        if (pp.deal && w.left == 0) return false;
        g.b = w.b;
        g.pair = w.pair;
        g.head = w.head;
        g.s = attn_seq(p, g.b, false);
        g.t0 = ap_tile(p, g.s, g.pair * AP_PAIR);
        g.t1 = ap_tile(p, g.s, g.pair * AP_PAIR + AP_TILE);
        const uint2 span = ap_span(g.t0, g.t1);
        g.jb = span.x;
        g.je = g.j1 = span.y;
        g.starts = g.whole = true;
        if (pp.deal) {
            // the item's cost lies before its blocks: a range that ends in it has none of them
            const uint32_t len = span.y - span.x, before = w.piece ? 0 : AP_ITEM_COST;
            const uint32_t cost = w.piece ? (len + w.piece - 1) / w.piece * w.piece : len + before;
            const uint32_t take = cost - w.off > w.left ? static_cast<uint32_t>(w.left) : cost - w.off;
            const uint32_t end = w.off + take;
            const uint32_t last = end > before ? end - before : 0;
            g.jb += w.off > before ? w.off - before : 0;
            g.je = span.x + (last < len ? last : len);
            g.starts = w.off <= before;
            g.whole = g.starts && end == cost;
            w.left -= take;
            w.off = 0;
            if (w.left && ++w.head == p.kv_heads) {
                w.head = 0;
                if (++w.pair == ap_pairs(p, g.s)) {
                    w.pair = 0;
                    do ++w.b;
                    while (ap_pairs(p, attn_seq(p, w.b, false)) == 0);
                }
            }
        }
    } while (g.jb == g.je);
    return true;
}

// ---- the kernel ---------------------------------------------------------------------

template <int DP, bool BF16>
__device__ __forceinline__ void ap_chunks(const CUtensorMap &map_k, const CUtensorMap &map_v, const APParams &pp,
                                          uint8_t *ap_smem_raw) {
    using L = APrompt<DP>;
    const AttnParams &p = pp.a;
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(ap_smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::OFF_BAR);
    uint64_t *q_full = bars, *q_empty = bars + 2, *s_full = bars + 4, *p_full = bars + 6, *o_done = bars + 8;
    uint64_t *drain = bars + 10, *s_free = bars + 12, *edge = bars + 13, *seg_full = bars + 14;
    uint64_t *seg_empty = seg_full + AP_SEG_SLOTS, *kv_full = seg_empty + AP_SEG_SLOTS, *kv_empty = kv_full + L::STAGES;
    // TMEM base, abort, pairs, then the CTA's first item: sequence, pair, head, cost before
    uint32_t *misc = reinterpret_cast<uint32_t *>(kv_empty + L::STAGES);
    APShared *segs = reinterpret_cast<APShared *>(smem + L::OFF_SEG);
    static_assert((14 + 2 * AP_SEG_SLOTS + 2 * L::STAGES) * 8 + 32 <= 512, "barriers outgrow their place");
    volatile uint32_t *abort_flag = misc + 1;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;

    // ---- this CTA's share -------------------------------------------------------------
    // where blocks are dealt out: the sequences that have pairs and their first ones, and
    // the cost before each pair, in the place of the keys
    uint32_t *seq_of = reinterpret_cast<uint32_t *>(smem + L::OFF_KV), *first_of = seq_of + AP_MAX_PAIRS;
    uint64_t *cost_before = reinterpret_cast<uint64_t *>(first_of + AP_MAX_PAIRS);
    if (warp == 0) {
        uint32_t total = 0, found = 0;
        for (uint32_t b0 = 0; b0 < p.seqs; b0 += 32) {
            const uint32_t b = b0 + lane;
            uint32_t n = b < p.seqs ? ap_pairs(p, attn_seq(p, b, blockIdx.x == 0)) : 0;
            uint32_t inc = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t t = __shfl_up_sync(0xFFFFFFFFu, inc, o);
                if (lane >= static_cast<uint32_t>(o)) inc += t;
            }
            // sequences that overlap in q may have more pairs than there are rows
            if (n && total + inc > pp.max_pairs) raise_device_status(p.status, FM_STATUS_INVALID_ARGUMENT);
            if (pp.deal) {
                const uint32_t has = __ballot_sync(0xFFFFFFFFu, n && total + inc <= pp.max_pairs);
                if (has >> lane & 1u) {
                    const uint32_t at = found + __popc(has & ((1u << lane) - 1u));
                    seq_of[at] = b;
                    first_of[at] = total + inc - n;
                }
                found += __popc(has);
                inc = has >> lane & 1u ? inc : 0; // the last pair that counts
                total = __reduce_max_sync(0xFFFFFFFFu, inc ? total + inc : total);
            } else {
                total += __shfl_sync(0xFFFFFFFFu, inc, 31);
            }
        }
        if (lane == 0) {
            misc[2] = total;
            misc[3] = found;
        }
    } else if (threadIdx.x == 32) {
        for (uint32_t i = 0; i < 2; ++i) {
            mbar_init(&q_full[i], 1);
            mbar_init(&q_empty[i], 1);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 128);
            mbar_init(&o_done[i], 1);
            mbar_init(&drain[i], 1);
        }
        for (uint32_t i = 0; i < AP_SEG_SLOTS; ++i) {
            mbar_init(&seg_full[i], 1);
            mbar_init(&seg_empty[i], AP_SEG_READERS);
        }
        mbar_init(s_free, 128);
        mbar_init(edge, 1);
        for (uint32_t i = 0; i < L::STAGES; ++i) {
            mbar_init(&kv_full[i], 1);
            mbar_init(&kv_empty[i], 1);
        }
        misc[1] = 0;
        fence_barrier_init();
    }
    __syncthreads();
    APWalk walk{};
    uint64_t per = 0;
    if (pp.deal) {
        const uint32_t pairs = misc[2], listed = misc[3];
        for (uint32_t i = threadIdx.x; i < pairs; i += AP_THREADS) {
            uint32_t lo = 0, hi = listed; // the last listed sequence whose first pair is not after i
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) / 2;
                if (first_of[mid] <= i)
                    lo = mid;
                else
                    hi = mid;
            }
            const AttnSeq s = attn_seq(p, seq_of[lo], false);
            const uint32_t row0 = (i - first_of[lo]) * AP_PAIR;
            const uint2 span = ap_span(ap_tile(p, s, row0), ap_tile(p, s, row0 + AP_TILE));
            cost_before[i + 1] = span.y - span.x;
        }
        __syncthreads();
        if (warp == 0) {
            uint32_t piece = 0;
            // pieces that the CTAs take of one head's items; sequences of few rows beside them keep
            // half of the SMs (chunks of 64 rows, 16 heads on one key head, behind 16000 keys beside 7
            // sequences 59 us, 65 without; of 300 behind 2000 beside one 44 and 40)
            const uint32_t budget = pp.ctas / (p.row_limit ? 2u : 1u) / p.kv_heads;
            if (pairs && pairs <= budget) {
                // the shortest pieces of which there are no more than CTAs
                uint32_t all = 0, longest = 0;
                for (uint32_t i = lane; i < pairs; i += 32) {
                    const uint32_t len = static_cast<uint32_t>(cost_before[i + 1]);
                    all += len;
                    longest = len > longest ? len : longest;
                }
                all = __reduce_add_sync(0xFFFFFFFFu, all);
                longest = __reduce_max_sync(0xFFFFFFFFu, longest);
                uint32_t lo = (all + budget - 1) / budget, hi = longest;
                while (lo < hi) {
                    const uint32_t mid = (lo + hi) / 2;
                    uint32_t n = 0;
                    for (uint32_t i = lane; i < pairs; i += 32)
                        n += (static_cast<uint32_t>(cost_before[i + 1]) + mid - 1) / mid;
                    if (__reduce_add_sync(0xFFFFFFFFu, n) <= budget)
                        hi = mid;
                    else
                        lo = mid + 1;
                }
                piece = lo < AP_LEAST_PIECE ? AP_LEAST_PIECE : lo;
                if (piece + AP_LEAST_SAVED > longest) piece = longest;
                // many CTAs idle: even ranges are shorter, with what a second item in them costs
                if (piece > all * p.kv_heads / pp.ctas + AP_LEAST_SAVED) piece = 0;
            }
            if (lane == 0) misc[0] = piece;
            uint64_t before = 0;
            for (uint32_t i0 = 0; i0 < pairs; i0 += 32) {
                uint64_t inc = i0 + lane < pairs ? cost_before[i0 + lane + 1] : 0;
                if (inc) inc = piece ? (static_cast<uint32_t>(inc) + piece - 1) / piece * piece : inc + AP_ITEM_COST;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint64_t t = __shfl_up_sync(0xFFFFFFFFu, inc, o);
                    if (lane >= static_cast<uint32_t>(o)) inc += t;
                }
                if (i0 + lane < pairs) cost_before[i0 + lane + 1] = before + inc;
                before += __shfl_sync(0xFFFFFFFFu, inc, 31);
            }
            if (lane == 0) cost_before[0] = 0;
        }
        __syncthreads();
        const uint64_t total = cost_before[pairs] * p.kv_heads, even = (total + pp.ctas - 1) / pp.ctas;
        walk.piece = misc[0];
        per = walk.piece ? walk.piece : even > AP_LEAST_COST ? even : AP_LEAST_COST;
        const uint64_t begin = blockIdx.x * per;
        if (threadIdx.x == 0) pp.tail[blockIdx.x] = make_int4(-1, 0, 0, 0);
        if (begin >= total) return;
        walk.left = total - begin < per ? total - begin : per;
        for (uint32_t i = threadIdx.x; i < pairs; i += AP_THREADS) {
            if (begin < cost_before[i] * p.kv_heads || begin >= cost_before[i + 1] * p.kv_heads) continue;
            uint32_t at = 0;
            while (at + 1 < listed && first_of[at + 1] <= i) ++at;
            const uint64_t inside = begin - cost_before[i] * p.kv_heads, n = cost_before[i + 1] - cost_before[i];
            misc[4] = seq_of[at];
            misc[5] = i - first_of[at];
            misc[6] = static_cast<uint32_t>(inside / n);
            misc[7] = static_cast<uint32_t>(inside % n);
        }
        __syncthreads();
        walk.b = misc[4];
        walk.pair = misc[5];
        walk.head = misc[6];
        walk.off = misc[7];
        fence_proxy_async(); // the copies of keys come into the tables' place
    } else {
        walk.left = static_cast<uint64_t>(misc[2]) * p.kv_heads;
        if (blockIdx.x >= walk.left) return;
    }

    if (warp == 11) {
        tmem_alloc(misc, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = misc[0];

    // Readers of segments: the k-th one, or false at the end.
    auto segment = [&](uint32_t k) -> const APShared * {
        if (!ap_wait(&seg_full[k % AP_SEG_SLOTS], (k / AP_SEG_SLOTS) & 1u, abort_flag, p.status)) return nullptr;
        const APShared *g = &segs[k % AP_SEG_SLOTS];
        return g->je ? g : nullptr;
    };
    auto release = [&](uint32_t k) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&seg_empty[k % AP_SEG_SLOTS]);
    };

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;\n");
        if (warp == 8) {
            // ---- the segments, their keys and values --------------------------------------
            const uint32_t R = pp.box_rows, n_boxes = AP_KEYS / R;
            uint32_t it = 0, edges = 0;
            bool going = true, more = true;
            APSeg g;
            for (uint32_t k = 0; going && more; ++k) {
                more = ap_next(pp, walk, g);
                going = ap_wait(&seg_empty[k % AP_SEG_SLOTS], ((k / AP_SEG_SLOTS) & 1u) ^ 1u, abort_flag, p.status);
                if (!going) break;
                const AttnSeq &s = g.s;
                if (lane == 0) {
                    APShared &o = segs[k % AP_SEG_SLOTS];
                    o.jb = g.jb;
                    o.je = more ? g.je : 0;
#pragma unroll
                    for (uint32_t t = 0; t < 2; ++t) {
                        const APTile &tile = t ? g.t1 : g.t0;
                        const uint32_t tb = tile.j0 > g.jb ? tile.j0 : g.jb, te = tile.j1 < g.je ? tile.j1 : g.je;
                        o.tb[t] = tb;
                        o.te[t] = te > tb ? te : tb;
                        o.whole_lo[t] = tile.whole_lo;
                        o.whole_hi[t] = tile.whole_hi;
                        o.rows[t] = tile.rows;
                    }
                    o.row0 = g.pair * AP_PAIR;
                    o.q0 = s.q0;
                    o.ql = s.ql;
                    o.kl = s.kl;
                    o.head = g.head;
                    o.starts = g.starts;
                    o.whole = g.whole;
                    mbar_arrive(&seg_full[k % AP_SEG_SLOTS]);
                    if (more && pp.deal && g.starts && g.je < g.j1) {
                        // the rest of the item goes to the next CTAs, `per` blocks each (to fewer
                        // than that takes where sequences overlap in q, which has been reported)
                        const uint64_t rest = g.j1 - g.je, most = pp.ctas - blockIdx.x;
                        const uint64_t parts = 1 + (rest + per - 1) / per;
                        pp.tail[blockIdx.x] = make_int4(static_cast<int>(g.b), static_cast<int>(g.pair),
                                                        static_cast<int>(g.head),
                                                        static_cast<int>(parts < most ? parts : most));
                    }
                }
                if (!more) break;
                for (uint32_t j = g.jb; j < g.je && going; ++j) {
                    const uint32_t key = j * AP_KEYS + lane * R;
                    const bool live = lane < n_boxes && key < s.kl && key + R > s.lo;
                    int32_t page = 0, row = 0;
                    if (live) {
                        const uint32_t at = key / p.page_size;
                        row = static_cast<int32_t>(key - at * p.page_size);
                        page = __ldg(p.table + g.b * p.tb + at);
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
                                            static_cast<int32_t>(h * 64), pp.heads_first ? static_cast<int32_t>(g.head) : row,
                                            pp.heads_first ? row : static_cast<int32_t>(g.head), page, bar);
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
            }
            // what was asked for must land before the CTA's shared memory goes away
            if (!going)
                for (uint32_t i = it > L::STAGES ? it - L::STAGES : 0; i < it; ++i)
                    (void)mbar_wait(&kv_full[i % L::STAGES], (i / L::STAGES) & 1u);
        } else if (warp == 11) {
            // ---- Q: a tile's 128 rows, a row by CH lanes, rows past the end as zeros ----------
            constexpr uint32_t CH = DP / 8, PER = 32 / CH;
            const uint32_t piece = lane % CH;
            uint32_t n[2] = {0, 0};
            const APShared *g;
            for (uint32_t k = 0; (g = segment(k)) != nullptr; ++k) {
                bool ok = true;
#pragma unroll
                for (uint32_t t = 0; t < 2; ++t) {
                    if (g->te[t] == g->tb[t] || !ok) continue;
                    ok = ap_wait(&q_empty[t], (n[t] & 1u) ^ 1u, abort_flag, p.status);
                    if (!ok) break;
                    ++n[t];
                    const uint32_t base = smem_u32(smem + t * L::BLOCK) + (piece >> 3) * L::HALF;
                    for (uint32_t r0 = 0; r0 < AP_TILE; r0 += 32) {
                        // the rows' places in q by their lanes, then handed to the lanes that copy
                        const uint32_t row = g->row0 + t * AP_TILE + r0 + lane, tok = row / p.group;
                        const int64_t at = tok < g->ql ? static_cast<int64_t>(
                                                             (static_cast<uint64_t>(g->q0) + tok) * p.qt +
                                                             (static_cast<uint64_t>(g->head) * p.group +
                                                              (row - tok * p.group)) * p.qh)
                                                       : -1;
#pragma unroll
                        for (uint32_t i = 0; i < 32 / PER; ++i) {
                            const int64_t from = __shfl_sync(0xFFFFFFFFu, at, i * PER + lane / CH);
                            const bool live = from >= 0 && piece * 8 < p.dim;
                            const uint32_t rr = r0 + i * PER + lane / CH;
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(
                                             base + rr * 128 + (((piece & 7u) ^ (rr & 7u)) << 4)),
                                         "l"(static_cast<const uint16_t *>(p.q) + (live ? from + piece * 8 : 0)),
                                         "r"(live ? 16u : 0u)
                                         : "memory");
                        }
                    }
                    cp_async_commit();
                    cp_async_wait<0>();
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&q_full[t]);
                }
                if (!ok) break;
                release(k);
            }
        } else {
            // ---- the products: warp 9 S = Q K^T, warp 10 O += P V, lane 0 of each ---------
            // S is asked for as soon as its place is free, so that it waits for its softmax
            // and not the other way round; the tensor cores take what is ready.
            const bool scores = warp == 9;
            constexpr uint32_t id_s = ap_idesc<BF16>(AP_KEYS, false), id_o = ap_idesc<BF16>(DP, true);
            uint32_t it = scores ? 0 : 1; // the next load of keys, or of values
            uint32_t n[2] = {0, 0}, q[2] = {0, 0}, s_used = 0;
            bool ok = true;
            const APShared *g;
            for (uint32_t k = 0; ok && (g = segment(k)) != nullptr; ++k) {
                const uint32_t jb = g->jb, je = g->je, tb[2] = {g->tb[0], g->tb[1]}, te[2] = {g->te[0], g->te[1]};
                release(k);
                for (uint32_t j = jb; j < je && ok; ++j, it += 2) {
                    const uint32_t st = it % L::STAGES;
                    const uint32_t kv = smem_u32(smem + L::OFF_KV + st * L::BLOCK);
                    ok = ap_wait(&kv_full[st], (it / L::STAGES) & 1u, abort_flag, p.status);
#pragma unroll
                    for (uint32_t t = 0; t < 2; ++t) {
                        if (!ok || j < tb[t] || j >= te[t]) continue;
                        if (scores) {
                            if (j == tb[t]) ok = ap_wait(&q_full[t], q[t]++ & 1u, abort_flag, p.status);
                            if (ok && s_used) ok = ap_wait(s_free, (s_used - 1) & 1u, abort_flag, p.status);
                            if (!ok) break;
                            tc_fence_after();
                            if (lane == 0) {
                                const uint32_t q_addr = smem_u32(smem + t * L::BLOCK);
#pragma unroll
                                for (uint32_t i = 0; i < DP / 16; ++i) {
                                    const uint32_t off = (i >> 2) * L::HALF + (i & 3u) * 32;
                                    mma_f16_ss(tmem + L::S_COL, smem_desc_sw128(q_addr + off),
                                               smem_desc_sw128(kv + off), id_s, i != 0);
                                }
                                tc_commit(&s_full[t]);
                                if (j + 1 == te[t]) tc_commit(&q_empty[t]);
                            }
                            ++s_used;
                        } else {
                            ok = ap_wait(&p_full[t], n[t] & 1u, abort_flag, p.status);
                            if (!ok) break;
                            tc_fence_after();
                            if (lane == 0) {
#pragma unroll
                                for (uint32_t i = 0; i < AP_KEYS / 16; ++i)
                                    mma_f16_ts(tmem + L::o_col(t), tmem + L::p_col(t) + i * 8,
                                               ap_desc_v(kv + i * 2048, L::HALF), id_o, i != 0 || j != tb[t]);
                                tc_commit(&o_done[t]);
                            }
                        }
                        ++n[t];
                    }
                    if (ok && lane == 0) tc_commit(&kv_empty[st]);
                }
            }
            // every product and commit must have ended before tensor and shared memory go away
            if (lane == 0) {
                tc_commit(&drain[scores ? 0 : 1]);
                (void)mbar_wait(&drain[scores ? 0 : 1], 0);
            }
            __syncwarp();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;\n");
        // ---- softmax: one thread a row ------------------------------------------------
        const uint32_t t = warp >> 2, r = threadIdx.x & 127u;
        const uint32_t lane_addr = ((warp & 3u) * 32u) << 16;
        const uint32_t s_tmem = tmem + L::S_COL + lane_addr;
        const uint32_t p_tmem = tmem + (t ? L::p_col(1) : L::p_col(0)) + lane_addr;
        const uint32_t o_tmem = tmem + (t ? L::o_col(1) : L::o_col(0)) + lane_addr;
        const uint64_t scale2 = pack_f32x2(p.scale_log2, p.scale_log2);
        uint32_t count = 0; // blocks of this tile so far
        bool ok = true;
        const APShared *g;
        for (uint32_t k = 0; ok && (g = segment(k)) != nullptr; ++k) {
            // of the segment, only what the loop and the result need is kept: registers
            const bool valid = r < g->rows[t], whole = g->whole;
            const uint32_t tb = g->tb[t], blocks = g->te[t] - tb;
            const uint32_t whole_lo = g->whole_lo[t], whole_hi = g->whole_hi[t];
            const uint32_t slot = (blockIdx.x * 2 + (g->starts ? 1 : 0)) * AP_PAIR + t * AP_TILE + r;
            const uint32_t row = g->row0 + t * AP_TILE + r, tok = row / p.group;
            uint32_t key_lo = 0, key_hi = g->kl;
            if (valid) {
                const int64_t pos = static_cast<int64_t>(g->kl) - g->ql + tok;
                const int64_t hi = p.causal ? pos + 1 : g->kl, lo = p.window ? pos - p.window + 1 : 0;
                key_hi = hi > 0 ? static_cast<uint32_t>(hi) : 0;
                key_lo = lo > 0 ? static_cast<uint32_t>(lo) : 0;
            }
            const uint64_t token = static_cast<uint64_t>(g->q0) + tok;
            const uint32_t qhead = g->head * p.group + (row - tok * p.group);
            const uint64_t out_at = token * p.ot + static_cast<uint64_t>(qhead) * p.oh;
            const uint32_t lse_at = static_cast<uint32_t>(token * p.heads) + qhead;
            release(k);
            float m = -INFINITY; // in log2
            uint64_t sums[4] = {0, 0, 0, 0}; // two f32 sums each
            for (uint32_t n = 0; n < blocks; ++n, ++count) {
                ok = ap_wait(&s_full[t], count & 1u, abort_flag, p.status);
                if (!ok) break;
                tc_fence_after();
                uint32_t x[4][32];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld32(s_tmem + c * 32, x[c]);
                tmem_wait_ld();
#pragma unroll
                for (int c = 0; c < 4; ++c) pin(x[c]);
                tc_fence_before();
                mbar_arrive(s_free);
                const uint32_t key0 = (tb + n) * AP_KEYS;
                if (key0 + AP_KEYS > whole_hi || key0 < whole_lo) {
                    // the row sees keys [gone, seen) of the block; most 32s are all or nothing to a warp
                    const uint32_t seen = key_hi > key0 ? key_hi - key0 : 0;
                    const uint32_t gone = key_lo > key0 ? key_lo - key0 : 0;
#pragma unroll
                    for (uint32_t c = 0; c < 4; ++c) {
                        if (!__any_sync(0xFFFFFFFFu, seen < c * 32 + 32 || gone > c * 32)) continue;
#pragma unroll
                        for (uint32_t i = 0; i < 32; ++i)
                            if (c * 32 + i - gone >= seen - gone) x[c][i] = 0xFF800000u; // -inf
                    }
                }
                float top[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    top[c] = __uint_as_float(x[c][0]);
#pragma unroll
                    for (int i = 1; i < 31; i += 2)
                        top[c] = max3(top[c], __uint_as_float(x[c][i]), __uint_as_float(x[c][i + 1]));
                    top[c] = max2(top[c], __uint_as_float(x[c][31]));
                }
                const float high = max2(max3(top[0], top[1], top[2]), top[3]) * p.scale_log2;
                if (__any_sync(0xFFFFFFFFu, !(high <= m + 8.0f))) {
                    const float to = max2(m, high);
                    const float f = m == -INFINITY ? 0.0f : exp2_approx(m - to);
                    m = to;
                    if (n) { // the last block's product has written O
                        ok = ap_wait(&o_done[t], (count - 1) & 1u, abort_flag, p.status);
                        if (!ok) break;
                        tc_fence_after();
                        const uint64_t f2 = pack_f32x2(f, f);
#pragma unroll
                        for (int i = 0; i < 4; ++i) sums[i] = fma_f32x2(sums[i], f2, 0);
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
                const float base = m == -INFINITY ? 0.0f : m - m - m; // NaN where m is or is infinite
                const uint64_t base2 = pack_f32x2(base, base);
                // all of the row's weights before the first store: the special-function unit runs on
                uint32_t w[2][32];
#pragma unroll
                for (int i = 0; i < 64; ++i) {
                    const uint32_t *e = &x[i >> 4][(i & 15) * 2];
                    float a, c2;
                    unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(e[0]), __uint_as_float(e[1])), scale2, base2), a, c2);
                    a = exp2_approx(a);
                    c2 = exp2_approx(c2);
                    sums[i & 3] = add_f32x2(sums[i & 3], pack_f32x2(a, c2));
                    w[i >> 5][i & 31] = pack_pair<BF16>(a, c2);
                }
                if (n) { // the last block's product has read P
                    ok = ap_wait(&o_done[t], (count - 1) & 1u, abort_flag, p.status);
                    tc_fence_after();
                }
                if (!ok) break;
                tmem_st32(p_tmem, w[0]);
                tmem_st32(p_tmem + 32, w[1]);
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(&p_full[t]);
            }
            // ---- result, while the next segment's first product runs ---------------------
            if (ok && blocks) ok = ap_wait(&o_done[t], (count - 1) & 1u, abort_flag, p.status);
            if (!ok || __ballot_sync(0xFFFFFFFFu, valid) == 0) continue;
            tc_fence_after();
            float a, c2;
            unpack_f32x2(add_f32x2(add_f32x2(sums[0], sums[1]), add_f32x2(sums[2], sums[3])), a, c2);
            const float sum = blocks ? a + c2 : 0.0f;
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            uint16_t *out = static_cast<uint16_t *>(p.out) + out_at;
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
                if (!valid) continue;
                if (whole) {
                    uint32_t v[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        v[i] = pack_pair<BF16>(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
#pragma unroll
                    for (uint32_t i = 0; i < 16; i += 8) {
                        const uint32_t col = c * 32u + i * 2;
                        if (pp.wide) {
                            if (col < p.dim) store_32b(out + col, &v[i]);
                            continue;
                        }
                        if (col < p.dim)
                            *reinterpret_cast<uint4 *>(out + col) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                        if (col + 8 < p.dim)
                            *reinterpret_cast<uint4 *>(out + col + 8) =
                                make_uint4(v[i + 4], v[i + 5], v[i + 6], v[i + 7]);
                    }
                } else {
                    float *dst = pp.part + static_cast<uint64_t>(slot) * DP + c * 32;
#pragma unroll
                    for (int i = 0; i < 32; i += 8) store_32b(dst + i, &o[i]);
                }
            }
            if (valid) {
                if (!whole)
                    pp.part_ml[slot] = make_float2(m, sum);
                else if (p.lse)
                    p.lse[lse_at] = sum == 0.0f ? -INFINITY : m * 0.6931471805599453f + logf(sum);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 11) tmem_dealloc(tmem, 512);
}

template <int DP, bool BF16>
__global__ void __launch_bounds__(AP_THREADS, 1)
    attn_prompt_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                       const __grid_constant__ APParams pp) {
    extern __shared__ __align__(1024) uint8_t ap_smem_raw[];
    // what follows on the stream may come to the SMs that have nothing to do here
    after_stream();
    let_next();
    ap_chunks<DP, BF16>(map_k, map_v, pp, ap_smem_raw);
}

template <int DP> constexpr uint32_t AP_BESIDE_SMEM = ARows<DP>::SMEM > APrompt<DP>::SMEM ? ARows<DP>::SMEM : APrompt<DP>::SMEM;

// Chunks, and beside them the sequences of few rows on the SMs that the chunks leave free: one
// grid, whose CTAs all wait for what came before it on the stream.  (As a launch of its own that
// began beside the chunks' the second part could not wait without running after the first.)  The
// first CTAs are the prompt kernel's; of the threads of the others two warpgroups work, with the
// third one's registers.  Measured, heads of 128, 8 key heads: a chunk of up to 512 behind 4000
// keys beside 31 decoding sequences 103 us, against 119 with one kernel after the other; of 510
// beside 7 with a window of 1000 keys (16 key heads) 44 against 65.
template <int DP, bool BF16>
__global__ void __launch_bounds__(AP_THREADS, 1)
    attn_beside_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                       const __grid_constant__ APParams pp) {
    extern __shared__ __align__(1024) uint8_t ap_smem_raw[];
    static_assert(AR_THREADS == 256, "two warpgroups");
    after_stream();
    let_next();
    if (blockIdx.x < pp.ctas) {
        ap_chunks<DP, BF16>(map_k, map_v, pp, ap_smem_raw);
        return;
    }
    if (threadIdx.x >= AR_THREADS) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;\n");
        return;
    }
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;\n");
    const uint32_t cta = blockIdx.x - pp.ctas, ctas = gridDim.x - pp.ctas;
    if (pp.rows_form == AR_CLUSTER)
        ar_cluster<DP, BF16>(pp.a, ap_smem_raw, cta, pp.rows_tiles);
    else if (pp.rows_form == AR_RANGES)
        ar_ranges<DP, BF16>(pp.a, ap_smem_raw, cta, ctas);
    else if (threadIdx.x < pp.rows_warps * 32)
        ar_unit<DP, BF16>(pp.a, ap_smem_raw, cta, ctas, pp.rows_tiles);
}

// Adds up the fragments of the items that were cut: blockIdx.x the CTA in which
// one begins, blockIdx.y sixteen of its rows, a warp a row.
constexpr uint32_t AJ_SLICES = 16;

template <int DP, bool BF16> __global__ void __launch_bounds__(256) attn_join_kernel(const __grid_constant__ APParams pp) {
    constexpr int V = DP / 32;
    const AttnParams &p = pp.a;
    after_stream();
    let_next();
    const int4 tail = pp.tail[blockIdx.x];
    if (tail.x < 0) return;
    const uint32_t lane = threadIdx.x & 31u;
    const AttnSeq s = attn_seq(p, static_cast<uint32_t>(tail.x), false);
    for (uint32_t k = threadIdx.x >> 5; k < AP_PAIR / AJ_SLICES; k += 8) {
        const uint32_t in = blockIdx.y * (AP_PAIR / AJ_SLICES) + k;
        const APRow w = ap_row(p, s, static_cast<uint32_t>(tail.z), static_cast<uint32_t>(tail.y), in / AP_TILE,
                               in % AP_TILE);
        if (!w.valid) continue;
        auto slot_of = [&](int i) { return ((blockIdx.x + i) * 2ull + (i == 0 ? 1 : 0)) * AP_PAIR + in; };
        float top = -INFINITY;
        for (int i = 0; i < tail.w; ++i) top = fmaxf(top, pp.part_ml[slot_of(i)].x);
        float acc[V] = {}, sum = 0.0f;
#pragma unroll 4
        for (int i = 0; i < tail.w; ++i) {
            const uint64_t slot = slot_of(i);
            const float2 ml = pp.part_ml[slot];
            const float f = ml.x == -INFINITY ? 0.0f : exp2_approx(ml.x - top);
            sum += ml.y * f;
#pragma unroll
            for (int x = 0; x < V; ++x) acc[x] += pp.part[slot * DP + lane * V + x] * f;
        }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        uint16_t *dst = static_cast<uint16_t *>(p.out) + w.token * p.ot + w.qhead * p.oh;
#pragma unroll
        for (int x = 0; x < V; x += 2)
            if (lane * V + x < p.dim)
                *reinterpret_cast<uint32_t *>(dst + lane * V + x) = pack_pair<BF16>(acc[x] * inv, acc[x + 1] * inv);
        if (p.lse && lane == 0)
            p.lse[w.token * p.heads + w.qhead] = sum == 0.0f ? -INFINITY : top * 0.6931471805599453f + logf(sum);
    }
}

} // namespace fmb
