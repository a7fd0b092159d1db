// attention_rows.cuh -- attention of few rows (decoding, short chunks) over a
// paged cache: one read of the keys and values, limited by HBM.
//
// The rows of a key head -- tokens x the query heads that share it -- make
// 16-row tiles, the M of mma.sync.m16n8k16; a step is 16 keys (32 of heads up to 64:
// with 16, a step's fixed work and not HBM set the pace, 125 us against 172 for twice
// the bytes): S = Q K^T (keys
// are the N), the running maximum and sum of the softmax, O += P V (keys are
// the K, P's accumulator fragments are its A fragments).  The contraction is
// far below what mma.sync does; the point is the stream of keys, so each warp
// has its own ring of 16-byte asynchronous copies in shared memory and waits
// for no other warp.  P is rounded to the cache's 16-bit type, as the matrix instruction
// takes it (the sums take it unrounded): for bf16 the result is within 0.0020 to 0.0024 of
// the 64-bit form (relative, as a norm), of which its own rounding is 0.0017.
//
// Work split: all (sequence, key head, row tile) units laid end to end, in
// steps of 16 keys, are cut into equal ranges, one a warp; whatever the lengths,
// every warp has the same work.  A unit counts for AR_UNIT_COST steps more than it has (its
// queries, its result): without that, 512 sequences of 2 to 1200 keys took 259 us, not 207,
// because some warps had dozens of units of a few keys.  A unit inside one range is written
// out at once; the fragments of a cut unit leave (O, max, sum) in f32 and
// attn_combine_kernel joins them, in order, so that the result does not depend
// on timing.  A warp has at most two fragments: of the unit that began before
// its range, and of the unit that goes on after it.
//
// Measured, 8 key heads of 128: 64 sequences of up to 8192 keys (1.09 GB) 170 to 181 us by
// machine, 94 to 99% of the rate of a copy; one sequence of 131071 keys and 4 key heads
// (268 MB) 55 us, of which the join of 1184 fragments takes 8.
#pragma once

#include "attention.cuh"
#include "tcgen05.cuh"

namespace fmb {

constexpr uint32_t AR_WARPS = 8, AR_THREADS = AR_WARPS * 32;
constexpr uint32_t AR_ROWS = 16, AR_MAX_CLUSTER = 8;
constexpr uint32_t AR_UNIT_COST = 2;
enum ARForm : uint32_t { AR_RANGES, AR_CLUSTER, AR_UNIT }; // see ar_ranges, ar_cluster, ar_unit
__host__ __device__ constexpr uint32_t ar_keys(int dp) { return dp == 64 ? 32 : 16; } // keys a step

template <int DP> struct ARows {
    static constexpr uint32_t ROW_BYTES = DP * 2;
    static constexpr uint32_t KEYS = ar_keys(DP);
    static constexpr uint32_t HALF = KEYS * ROW_BYTES; // K or V of a step
    static constexpr uint32_t STAGE = 2 * HALF;
    static constexpr uint32_t STAGES = 24576 / STAGE; // 24 KB a warp
    static constexpr uint32_t RINGS = AR_WARPS * STAGES * STAGE;
    static constexpr uint32_t SMEM = RINGS + 2048; // and what the warps tell each other
};

// Row tiles and steps a unit of sequence s in the rows kernel (no tiles: not its work).
struct ARShape {
    uint32_t tiles, step0, steps;
};
template <int DP> __device__ __forceinline__ ARShape ar_shape(const AttnParams &p, const AttnSeq &s) {
    constexpr uint32_t KEYS = ar_keys(DP);
    ARShape r;
    const uint64_t rows = static_cast<uint64_t>(s.ql) * p.group;
    r.tiles = rows <= p.row_limit ? static_cast<uint32_t>((rows + AR_ROWS - 1) / AR_ROWS) : 0;
    r.step0 = s.lo / KEYS;
    const uint32_t last = (s.kl + KEYS - 1) / KEYS;
    r.steps = last > r.step0 ? last - r.step0 : 1; // a unit without keys still writes its zeros
    return r;
}
// The sequence's place in the laid-out work; its units are `steps` + AR_UNIT_COST long, the cost first.
__device__ __forceinline__ uint64_t ar_length(const AttnParams &p, const ARShape &sh) {
    return static_cast<uint64_t>(sh.tiles) * p.kv_heads * (sh.steps + AR_UNIT_COST);
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

template <bool BF16>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, "
                     "%9}, {%0, %1, %2, %3};\n"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, "
                     "%9}, {%0, %1, %2, %3};\n"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The three forms below are device functions of CTA `cta` of `ctas` with 256 threads and shared
// memory at `smem`: kernels of their own, or a part of the grid of attn_beside_kernel, whose
// other CTAs take the chunks.

// A place in the laid-out work.
struct ARCursor {
    uint32_t b, tile, step; // tile: key head * row tiles + row tile
    uint32_t at;            // from the range's begin
    AttnSeq s;
    ARShape sh;
};

template <int DP> __device__ __forceinline__ void ar_enter(const AttnParams &p, ARCursor &c) {
    // the next sequence that has tiles; the caller stops at the range's end before there is none
    while (c.b < p.seqs) {
        c.s = attn_seq(p, c.b, false);
        c.sh = ar_shape<DP>(p, c.s);
        if (c.sh.tiles) return;
        ++c.b;
    }
}

template <int DP> __device__ __forceinline__ void ar_advance(const AttnParams &p, ARCursor &c) {
    ++c.at;
    if (++c.step < c.sh.steps) return;
    c.step = 0;
    c.at += AR_UNIT_COST;
    if (++c.tile < c.sh.tiles * p.kv_heads) return;
    c.tile = 0;
    ++c.b;
    ar_enter<DP>(p, c);
}

// Queues the copies of a step's keys and values; what is not to be read becomes zeros.
template <int DP>
__device__ __forceinline__ void ar_fetch(const AttnParams &p, uint32_t stage, int64_t offset, uint32_t lane) {
    constexpr uint32_t CH = DP / 8, PER = 32 / CH; // 16-byte pieces a row, rows a round
    const uint32_t piece = lane % CH;
#pragma unroll
    for (uint32_t i = 0; i < ARows<DP>::KEYS / PER; ++i) {
        const uint32_t row = i * PER + lane / CH;
        const int64_t at = __shfl_sync(0xFFFFFFFFu, offset, row);
        const bool live = at >= 0 && piece * 8 < p.dim;
        const int64_t from = live ? at + piece * 8 : 0;
        const uint32_t dst = stage + row * ARows<DP>::ROW_BYTES + ((piece ^ (row & 7u)) << 4);
        const uint32_t n = live ? 16u : 0u;
        asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;\n" ::"r"(dst),
                     "l"(static_cast<const uint16_t *>(p.kc) + from), "r"(n)
                     : "memory");
        asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;\n" ::"r"(dst + ARows<DP>::HALF),
                     "l"(static_cast<const uint16_t *>(p.vc) + from), "r"(n)
                     : "memory");
    }
}

// Exclusive sum over the CTA of one 64-bit value a thread; *total: of all.
__device__ __forceinline__ uint64_t ar_block_scan(uint64_t v, uint64_t *s_part, uint64_t *total) {
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    uint64_t inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t t = __shfl_up_sync(0xFFFFFFFFu, inc, o);
        if (lane >= static_cast<uint32_t>(o)) inc += t;
    }
    __syncthreads();
    if (lane == 31) s_part[warp] = inc;
    __syncthreads();
    uint64_t before = 0, all = 0;
#pragma unroll
    for (uint32_t w = 0; w < AR_WARPS; ++w) {
        if (w < warp) before += s_part[w];
        all += s_part[w];
    }
    *total = all;
    return before + inc - v;
}

// A warp's 16 rows of a unit: Q fragments, O, and of rows lane / 4 and lane / 4 + 8 the
// reference exponent (in log2), the lane's part of the sum, and the keys that the row sees.
template <int DP, bool BF16> struct ARState {
    uint32_t qf[DP / 16][4];
    float o[DP / 8][4];
    float m[2], l[2];
    uint32_t key_lo[2], key_hi[2];

    __device__ __forceinline__ void begin(const AttnParams &p, const AttnSeq &s, uint32_t head, uint32_t rt,
                                          uint32_t lane) {
        const uint16_t *rows[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const uint32_t row = rt * AR_ROWS + lane / 4 + r * 8;
            const uint32_t t = row / p.group, g = row - t * p.group;
            m[r] = -INFINITY;
            l[r] = 0.0f;
            key_lo[r] = key_hi[r] = 0;
            rows[r] = nullptr;
            if (t < s.ql) {
                const int64_t pos = static_cast<int64_t>(s.kl) - s.ql + t;
                const int64_t hi = p.causal ? pos + 1 : s.kl;
                const int64_t lo = p.window ? pos - p.window + 1 : 0;
                key_hi[r] = hi > 0 ? static_cast<uint32_t>(hi) : 0;
                key_lo[r] = lo > 0 ? static_cast<uint32_t>(lo) : 0;
                rows[r] = static_cast<const uint16_t *>(p.q) + (static_cast<uint64_t>(s.q0) + t) * p.qt +
                          static_cast<int64_t>(head * p.group + g) * p.qh;
            }
        }
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const uint32_t col = k * 16 + (x >> 1) * 8 + (lane & 3u) * 2;
                const uint16_t *row = rows[x & 1];
                qf[k][x] = row && col < p.dim ? *reinterpret_cast<const uint32_t *>(row + col) : 0u;
            }
#pragma unroll
        for (int n = 0; n < DP / 8; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[n][x] = 0.0f;
    }

    // The keys and values of stage `st`, the first of them key `key_first`.
    __device__ __forceinline__ void step(const AttnParams &p, uint32_t st, uint32_t key_first, uint32_t lane) {
        using L = ARows<DP>;
        constexpr int N = L::KEYS / 8; // 8-key tiles
        // S = Q K^T
        float sc[N][4] = {};
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
#pragma unroll
            for (int n = 0; n < N; n += 2) {
                uint32_t b[4];
                const uint32_t row = n * 8 + ((lane >> 4) << 3) + (lane & 7u), piece = k * 2 + ((lane >> 3) & 1u);
                ldsm4(st + row * L::ROW_BYTES + ((piece ^ (row & 7u)) << 4), b);
                mma_16816<BF16>(sc[n], qf[k], b[0], b[1]);
                mma_16816<BF16>(sc[n + 1], qf[k], b[2], b[3]);
            }
        }
        const uint32_t key0 = key_first + (lane & 3u) * 2;
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int r = x >> 1;
                const uint32_t key = key0 + n * 8 + (x & 1);
                sc[n][x] = key >= key_lo[r] && key < key_hi[r] ? sc[n][x] * p.scale_log2 : -INFINITY;
                top[r] = fmaxf(top[r], sc[n][x]);
            }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            top[r] = fmaxf(top[r], __shfl_xor_sync(0xFFFFFFFFu, top[r], 1));
            top[r] = fmaxf(top[r], __shfl_xor_sync(0xFFFFFFFFu, top[r], 2));
        }
        // the reference exponent moves only when it is over 2^8 too small: the weights
        // stay in range of f32 sums and of 16-bit products, and O is rarely rescaled
        if (__any_sync(0xFFFFFFFFu, top[0] > m[0] + 8.0f || top[1] > m[1] + 8.0f)) {
            float f2[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float to = fmaxf(m[r], top[r]);
                f2[r] = m[r] == -INFINITY ? 0.0f : exp2_approx(m[r] - to);
                m[r] = to;
                l[r] *= f2[r];
            }
#pragma unroll
            for (int n = 0; n < DP / 8; ++n)
#pragma unroll
                for (int x = 0; x < 4; ++x) o[n][x] *= f2[x >> 1];
        }
        const float base[2] = {m[0] == -INFINITY ? 0.0f : m[0], m[1] == -INFINITY ? 0.0f : m[1]};
        uint32_t pf[N / 2][4];
#pragma unroll
        for (int n = 0; n < N; ++n) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                sc[n][x] = exp2_approx(sc[n][x] - base[x >> 1]);
                l[x >> 1] += sc[n][x];
            }
            pf[n / 2][2 * (n & 1)] = pack_pair<BF16>(sc[n][0], sc[n][1]);
            pf[n / 2][2 * (n & 1) + 1] = pack_pair<BF16>(sc[n][2], sc[n][3]);
        }
        // O += P V
#pragma unroll
        for (int k = 0; k < N / 2; ++k)
#pragma unroll
            for (int n = 0; n < DP / 16; ++n) {
                uint32_t b[4];
                const uint32_t row = k * 16 + (((lane >> 3) & 1u) << 3) + (lane & 7u), piece = n * 2 + (lane >> 4);
                ldsm4_t(st + L::HALF + row * L::ROW_BYTES + ((piece ^ (row & 7u)) << 4), b);
                mma_16816<BF16>(o[2 * n], pf[k], b[0], b[1]);
                mma_16816<BF16>(o[2 * n + 1], pf[k], b[2], b[3]);
            }
    }

    // The rows' sums, in every lane of a row's four.
    __device__ __forceinline__ float sum(int r) const {
        float v = l[r];
        v += __shfl_xor_sync(0xFFFFFFFFu, v, 1);
        return v + __shfl_xor_sync(0xFFFFFFFFu, v, 2);
    }
};

// A cache row's place: the offset of the lane's key (lane modulo the keys of a step) from
// `key_first` on, or -1: not to be read.
template <int DP> __device__ __forceinline__ int64_t ar_key_at(const AttnParams &p, const AttnSeq &s, uint32_t b, uint32_t head,
                                             uint32_t key_first, uint32_t lane) {
    const uint32_t key = key_first + (lane & (ar_keys(DP) - 1));
    if (key < s.lo || key >= s.kl) return -1;
    const uint32_t page = key / p.page_size;
    const int32_t id = __ldg(p.table + b * p.tb + page);
    if (id < 0 || static_cast<uint32_t>(id) >= p.n_pages) {
        raise_device_status(p.status, FM_STATUS_INVALID_ARGUMENT);
        return -1;
    }
    return id * p.cp + static_cast<int64_t>(key - page * p.page_size) * p.cr + head * p.ch;
}

// The result of row r of the lane's two, row `row` of the sequence and key head.
template <int DP, bool BF16>
__device__ __forceinline__ void ar_store_row(const AttnParams &p, const AttnSeq &s, uint32_t head, uint32_t row,
                                             const ARState<DP, BF16> &u, int r, float sum, uint32_t lane) {
    const uint32_t t = row / p.group, g = row - t * p.group;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const uint64_t h = head * p.group + g, token = static_cast<uint64_t>(s.q0) + t;
    uint16_t *dst = static_cast<uint16_t *>(p.out) + token * p.ot + h * p.oh;
#pragma unroll
    for (int n = 0; n < DP / 8; ++n) {
        const uint32_t col = n * 8 + (lane & 3u) * 2;
        if (col < p.dim)
            *reinterpret_cast<uint32_t *>(dst + col) = pack_pair<BF16>(u.o[n][2 * r] * inv, u.o[n][2 * r + 1] * inv);
    }
    if (p.lse && (lane & 3u) == 0)
        p.lse[token * p.heads + h] = sum == 0.0f ? -INFINITY : u.m[r] * 0.6931471805599453f + logf(sum);
}

template <int DP, bool BF16>
__device__ __forceinline__ void ar_ranges(const AttnParams &p, uint8_t *smem, uint32_t cta, uint32_t ctas) {
    using L = ARows<DP>;
    uint64_t *s_part = reinterpret_cast<uint64_t *>(smem + L::RINGS), *s_first = s_part + AR_WARPS;
    uint32_t *s_seq = reinterpret_cast<uint32_t *>(s_first + AR_WARPS);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;

    // ---- this warp's range, and the sequence that it begins in -------------------
    uint64_t total = 0, mine = 0, before = 0;
    const bool few = p.seqs <= AR_THREADS;
    for (uint32_t b0 = 0; b0 < p.seqs; b0 += AR_THREADS) {
        const uint32_t b = b0 + threadIdx.x;
        mine = 0;
        if (b < p.seqs) {
            const AttnSeq s = attn_seq(p, b, cta == 0);
            const ARShape sh = ar_shape<DP>(p, s);
            mine = ar_length(p, sh);
        }
        uint64_t sum;
        before = ar_block_scan(mine, s_part, &sum);
        if (cta == 0 && b < p.seqs) p.prefix[b] = total + before;
        total += sum;
    }
    if (cta == 0 && threadIdx.x == 0) p.prefix[p.seqs] = total;
    const uint64_t even = quotient(total + p.workers - 1, p.workers);
    const uint64_t per = even > p.least ? even : p.least;
    uint64_t running = 0;
    for (uint32_t b0 = 0; b0 < p.seqs; b0 += AR_THREADS) {
        const uint32_t b = b0 + threadIdx.x;
        if (!few) {
            mine = 0;
            if (b < p.seqs) {
                const AttnSeq s = attn_seq(p, b, false);
                const ARShape sh = ar_shape<DP>(p, s);
                mine = ar_length(p, sh);
            }
            uint64_t sum;
            before = running + ar_block_scan(mine, s_part, &sum);
            running += sum;
        }
        if (mine) {
#pragma unroll
            for (uint32_t w = 0; w < AR_WARPS; ++w) {
                const uint64_t at = (static_cast<uint64_t>(w) * ctas + cta) * per;
                if (at >= before && at < before + mine) {
                    s_seq[w] = b;
                    s_first[w] = before;
                }
            }
        }
    }
    __syncthreads();
    const uint64_t worker = static_cast<uint64_t>(warp) * ctas + cta;
    const uint64_t begin = worker * per;
    int4 tail = make_int4(-1, 0, 0, 0); // the unit that begins here and goes on after the range
    if (begin >= total) {
        if (lane == 0) p.tail_rows[worker] = tail;
        return;
    }
    const uint32_t end = static_cast<uint32_t>((total - begin < per) ? total - begin : per);

    ARCursor c;
    c.b = s_seq[warp];
    c.s = attn_seq(p, c.b, false);
    c.sh = ar_shape<DP>(p, c.s);
    const uint64_t inside = begin - s_first[warp];
    const uint32_t unit = c.sh.steps + AR_UNIT_COST;
    c.tile = static_cast<uint32_t>(quotient(inside, unit));
    const uint32_t in_unit = static_cast<uint32_t>(inside - static_cast<uint64_t>(c.tile) * unit);
    c.step = in_unit > AR_UNIT_COST ? in_unit - AR_UNIT_COST : 0;
    c.at = in_unit < AR_UNIT_COST ? AR_UNIT_COST - in_unit : 0;

    // ---- the stream of keys -------------------------------------------------------
    const uint32_t ring = smem_u32(smem) + warp * (L::STAGES * L::STAGE);
    ARCursor f = c;
    ARState<DP, BF16> u;
    uint32_t first_step = c.step;
    bool fresh = false;
    uint32_t fetched = 0;
    auto place = [&] { return ar_key_at<DP>(p, f.s, f.b, f.tile / f.sh.tiles, (f.sh.step0 + f.step) * L::KEYS, lane); };
    int64_t next = c.at < end ? place() : -1; // one step ahead of the copies: hides the table's latency
    if (c.at < end) u.begin(p, c.s, c.tile / c.sh.tiles, c.tile % c.sh.tiles, lane); // its loads before the keys'
    auto fetch = [&] {
        if (f.at < end) {
            ar_fetch<DP>(p, ring + (fetched % L::STAGES) * L::STAGE, next, lane);
            ++fetched;
            ar_advance<DP>(p, f);
            if (f.at < end) next = place();
        }
        cp_async_commit();
    };
#pragma unroll
    for (uint32_t i = 0; i + 1 < L::STAGES; ++i) fetch();

    for (uint32_t i = 0; c.at < end; ++i) {
        const uint32_t head = c.tile / c.sh.tiles, rt = c.tile - head * c.sh.tiles;
        if (fresh) {
            fresh = false;
            first_step = c.step;
            u.begin(p, c.s, head, rt, lane);
        }
        cp_async_wait<L::STAGES - 2>();
        __syncwarp();
        u.step(p, ring + (i % L::STAGES) * L::STAGE, (c.sh.step0 + c.step) * L::KEYS, lane);
        __syncwarp(); // every lane has read the stage that the next copies fill
        fetch();

        const bool done = c.step + 1 == c.sh.steps;
        if (done || c.at + 1 == end) {
            fresh = true;
            const bool whole = first_step == 0 && done;
            if (first_step == 0 && !done) {
                const uint64_t last = static_cast<uint64_t>(c.at) + (c.sh.steps - 1 - c.step);
                tail = make_int4(static_cast<int>(c.b), static_cast<int>(c.tile),
                                 static_cast<int>(quotient(last, per)) + 1, 0);
            }
            const uint64_t slot = worker * 2 + (first_step == 0 ? 1 : 0);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float sum = u.sum(r);
                const uint32_t in = lane / 4 + r * 8, row = rt * AR_ROWS + in;
                if (row >= c.s.ql * p.group) continue;
                if (whole) {
                    ar_store_row<DP, BF16>(p, c.s, head, row, u, r, sum, lane);
                } else {
                    float *dst = p.part + (slot * AR_ROWS + in) * DP;
#pragma unroll
                    for (int n = 0; n < DP / 8; ++n)
                        *reinterpret_cast<float2 *>(dst + n * 8 + (lane & 3u) * 2) =
                            make_float2(u.o[n][2 * r], u.o[n][2 * r + 1]);
                    if ((lane & 3u) == 0) p.part_ml[slot * AR_ROWS + in] = make_float2(u.m[r], sum);
                }
            }
        }
        ar_advance<DP>(p, c);
    }
    if (lane == 0) p.tail_rows[worker] = tail;
    cp_async_wait<0>();
}

template <int DP, bool BF16>
__global__ void __launch_bounds__(AR_THREADS, 1) attn_rows_kernel(const AttnParams p) {
    extern __shared__ __align__(1024) uint8_t ar_smem[];
    after_stream();
    let_next();
    ar_ranges<DP, BF16>(p, ar_smem, blockIdx.x, gridDim.x);
}

// ---- few units of short sequences: a cluster each ----------------------------------
//
// Where a cluster of CTAs a unit is all the GPU can do with the work (one short
// sequence, say), the unit's steps are cut over the cluster's warps, a CTA's
// warps are joined in its shared memory and the CTAs through each other's: one
// launch, no fragments in global memory.  blockIdx.x / cluster size: (sequence,
// key head, row tile), `unit_tiles` row tiles a sequence and head.
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_nctarank;\n" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// A value of CTA `rank`'s shared memory, at the address that `addr` has in this one's.
__device__ __forceinline__ float cluster_load(uint32_t addr, uint32_t rank) {
    uint32_t at;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(at) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(v) : "r"(at) : "memory");
    return v;
}

template <int DP, bool BF16>
__device__ __forceinline__ void ar_cluster(const AttnParams &p, uint8_t *smem, uint32_t cta, uint32_t unit_tiles) {
    using L = ARows<DP>;
    float(*s_m)[AR_ROWS] = reinterpret_cast<float(*)[AR_ROWS]>(smem + L::RINGS), (*s_l)[AR_ROWS] = s_m + AR_WARPS; // of the warps
    float *s_top = s_l[AR_WARPS], *s_sum = s_top + AR_ROWS;                                                      // of the CTA
    static_assert((2 * AR_WARPS + 2) * AR_ROWS * 4 <= L::SMEM - L::RINGS, "the sums outgrow their place");
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint32_t rank = cluster_rank(), ranks = cluster_size();
    const uint32_t unit = cta / ranks, rt = unit % unit_tiles;
    const uint32_t head = unit / unit_tiles % p.kv_heads, b = unit / unit_tiles / p.kv_heads;
    const AttnSeq s = attn_seq(p, b, threadIdx.x == 0 && rank == 0 && rt == 0 && head == 0);
    const ARShape sh = ar_shape<DP>(p, s);
    if (rt >= sh.tiles) return; // the whole cluster

    const uint32_t part = rank * AR_WARPS + warp, parts = ranks * AR_WARPS;
    const uint32_t begin = static_cast<uint32_t>(static_cast<uint64_t>(sh.steps) * part / parts);
    const uint32_t count = static_cast<uint32_t>(static_cast<uint64_t>(sh.steps) * (part + 1) / parts) - begin;
    const uint32_t key_first = (sh.step0 + begin) * L::KEYS;
    const uint32_t ring = smem_u32(smem) + warp * (L::STAGES * L::STAGE);
    uint32_t fetched = 0;
    int64_t next = count ? ar_key_at<DP>(p, s, b, head, key_first, lane) : -1;
    auto fetch = [&] {
        if (fetched < count) {
            ar_fetch<DP>(p, ring + (fetched % L::STAGES) * L::STAGE, next, lane);
            if (++fetched < count) next = ar_key_at<DP>(p, s, b, head, key_first + fetched * L::KEYS, lane);
        }
        cp_async_commit();
    };
#pragma unroll
    for (uint32_t i = 0; i + 1 < L::STAGES; ++i) fetch();
    ARState<DP, BF16> u;
    u.begin(p, s, head, rt, lane);
    for (uint32_t i = 0; i < count; ++i) {
        cp_async_wait<L::STAGES - 2>();
        __syncwarp();
        u.step(p, ring + (i % L::STAGES) * L::STAGE, key_first + i * L::KEYS, lane);
        __syncwarp();
        fetch();
    }
    cp_async_wait<0>();
    __syncwarp();
    // the warp's O over its ring, rows of DP
    const uint32_t all = s.ql * p.group - rt * AR_ROWS, rows = all < AR_ROWS ? all : AR_ROWS;
    float *mine = reinterpret_cast<float *>(smem + warp * (L::STAGES * L::STAGE));
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const float sum = u.sum(r);
        const uint32_t in = lane / 4 + r * 8;
        if (in >= rows) continue;
#pragma unroll
        for (int n = 0; n < DP / 8; ++n)
            *reinterpret_cast<float2 *>(mine + in * DP + n * 8 + (lane & 3u) * 2) =
                make_float2(u.o[n][2 * r], u.o[n][2 * r + 1]);
        if ((lane & 3u) == 0) {
            s_m[warp][in] = u.m[r];
            s_l[warp][in] = sum;
        }
    }
    __syncthreads();
    // the CTA's O behind warp 0's
    float *joined = reinterpret_cast<float *>(smem) + AR_ROWS * DP;
    for (uint32_t i = threadIdx.x; i < rows * DP; i += AR_THREADS) {
        const uint32_t in = i / DP;
        float top = -INFINITY, acc = 0.0f, sum = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < AR_WARPS; ++w) top = fmaxf(top, s_m[w][in]);
#pragma unroll
        for (uint32_t w = 0; w < AR_WARPS; ++w) {
            const float f = s_m[w][in] == -INFINITY ? 0.0f : exp2_approx(s_m[w][in] - top);
            sum += s_l[w][in] * f;
            acc += reinterpret_cast<const float *>(smem + w * (L::STAGES * L::STAGE))[i] * f;
        }
        joined[i] = acc;
        if (i % DP == 0) {
            s_top[in] = top;
            s_sum[in] = sum;
        }
    }
    cluster_sync();
    // rows rank, rank + ranks, ... of the unit
    const uint32_t top_at = smem_u32(s_top), sum_at = smem_u32(s_sum), o_at = smem_u32(joined);
    for (uint32_t i = threadIdx.x; i < AR_ROWS / ranks * (DP / 2); i += AR_THREADS) {
        const uint32_t in = i / (DP / 2) * ranks + rank, col = i % (DP / 2) * 2;
        if (in >= rows || col >= p.dim) continue;
        const uint32_t row = rt * AR_ROWS + in, t = row / p.group, g = row - t * p.group;
        // all CTAs' values under way together
        float m[AR_MAX_CLUSTER], l[AR_MAX_CLUSTER], v0[AR_MAX_CLUSTER], v1[AR_MAX_CLUSTER];
#pragma unroll
        for (uint32_t k = 0; k < AR_MAX_CLUSTER; ++k) {
            m[k] = -INFINITY;
            l[k] = v0[k] = v1[k] = 0.0f;
            if (k >= ranks) continue;
            m[k] = cluster_load(top_at + in * 4, k);
            l[k] = cluster_load(sum_at + in * 4, k);
            v0[k] = cluster_load(o_at + (in * DP + col) * 4, k);
            v1[k] = cluster_load(o_at + (in * DP + col) * 4 + 4, k);
        }
        float top = -INFINITY, sum = 0.0f, a0 = 0.0f, a1 = 0.0f;
#pragma unroll
        for (uint32_t k = 0; k < AR_MAX_CLUSTER; ++k) top = fmaxf(top, m[k]);
#pragma unroll
        for (uint32_t k = 0; k < AR_MAX_CLUSTER; ++k) {
            const float f = m[k] == -INFINITY ? 0.0f : exp2_approx(m[k] - top);
            sum += l[k] * f;
            a0 += v0[k] * f;
            a1 += v1[k] * f;
        }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        const uint64_t h = head * p.group + g, token = static_cast<uint64_t>(s.q0) + t;
        *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(p.out) + token * p.ot + h * p.oh + col) =
            pack_pair<BF16>(a0 * inv, a1 * inv);
        if (p.lse && col == 0)
            p.lse[token * p.heads + h] = sum == 0.0f ? -INFINITY : top * 0.6931471805599453f + logf(sum);
    }
    cluster_sync(); // nobody leaves while its shared memory is read
}

template <int DP, bool BF16>
__global__ void __launch_bounds__(AR_THREADS, 1) attn_cluster_kernel(const AttnParams p, uint32_t unit_tiles) {
    extern __shared__ __align__(1024) uint8_t ar_smem[];
    after_stream();
    let_next();
    ar_cluster<DP, BF16>(p, ar_smem, blockIdx.x, unit_tiles);
}

// ---- many units of very short sequences: a warp each ------------------------------
//
// Where a unit has few steps, reading is soon done and what is around it counts: the
// warps of a CTA take a unit each, from its first key to its last, and write its rows.
// No sums over the sequences to find the work, no fragments, one launch.
template <int DP, bool BF16>
__device__ __forceinline__ void ar_unit(const AttnParams &p, uint8_t *smem, uint32_t cta, uint32_t ctas, uint32_t unit_tiles) {
    using L = ARows<DP>;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint32_t unit = warp * ctas + cta, rt = unit % unit_tiles;
    const uint32_t head = unit / unit_tiles % p.kv_heads, b = unit / unit_tiles / p.kv_heads;
    if (b < p.seqs) {
        const AttnSeq s = attn_seq(p, b, lane == 0 && rt == 0 && head == 0);
        const ARShape sh = ar_shape<DP>(p, s);
        if (rt < sh.tiles) {
            const uint32_t ring = smem_u32(smem) + warp * (L::STAGES * L::STAGE), key_first = sh.step0 * L::KEYS;
            ARState<DP, BF16> u;
            uint32_t fetched = 0;
            int64_t next = ar_key_at<DP>(p, s, b, head, key_first, lane);
            u.begin(p, s, head, rt, lane); // its loads before the keys'
            auto fetch = [&] {
                if (fetched < sh.steps) {
                    ar_fetch<DP>(p, ring + (fetched % L::STAGES) * L::STAGE, next, lane);
                    if (++fetched < sh.steps) next = ar_key_at<DP>(p, s, b, head, key_first + fetched * L::KEYS, lane);
                }
                cp_async_commit();
            };
#pragma unroll
            for (uint32_t i = 0; i + 1 < L::STAGES; ++i) fetch();
            for (uint32_t i = 0; i < sh.steps; ++i) {
                cp_async_wait<L::STAGES - 2>();
                __syncwarp();
                u.step(p, ring + (i % L::STAGES) * L::STAGE, key_first + i * L::KEYS, lane);
                __syncwarp();
                fetch();
            }
            cp_async_wait<0>();
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float sum = u.sum(r);
                const uint32_t row = rt * AR_ROWS + lane / 4 + r * 8;
                if (row < s.ql * p.group) ar_store_row<DP, BF16>(p, s, head, row, u, r, sum, lane);
            }
        }
    }
}

template <int DP, bool BF16>
__global__ void __launch_bounds__(AR_THREADS, 1) attn_unit_kernel(const AttnParams p, uint32_t unit_tiles) {
    extern __shared__ __align__(1024) uint8_t ar_smem[];
    after_stream();
    let_next();
    ar_unit<DP, BF16>(p, ar_smem, blockIdx.x, gridDim.x, unit_tiles);
}

// Joins the fragments of the units that were cut.  A CTA of W warps takes a row (one of C
// parts of it, so that few rows keep more SMs busy) of a unit: of unit blockIdx.x, or, where
// there are more units than warps in the rows kernel, of the unit that was cut at the end of
// warp blockIdx.x's range.  Warp i takes fragments
// i, i + W, ..., a lane DP / 32 / C values of the head, with the loads of F fragments under
// way together.
template <int DP, bool BF16, int W, int F, int C>
__global__ void __launch_bounds__(W * 32) attn_combine_kernel(const AttnParams p, bool by_worker) {
    constexpr int V = DP / 32 / C;
    __shared__ float s_o[W][DP / C];
    __shared__ float s_m[W], s_l[W];
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    after_stream();
    let_next();
    const uint32_t y = blockIdx.y / C, col0 = blockIdx.y % C * (DP / C);
    AttnSeq s;
    uint32_t head, row, n;
    uint64_t w0;
    if (by_worker) {
        const int4 tail = p.tail_rows[blockIdx.x];
        if (tail.x < 0) return;
        s = attn_seq(p, static_cast<uint32_t>(tail.x), false);
        const ARShape sh = ar_shape<DP>(p, s);
        const uint32_t tile = static_cast<uint32_t>(tail.y);
        head = tile / sh.tiles;
        row = (tile - head * sh.tiles) * AR_ROWS + y;
        n = static_cast<uint32_t>(tail.z);
        w0 = blockIdx.x;
        if (row >= s.ql * p.group) return;
    } else {
        const uint32_t b = blockIdx.x / p.kv_heads;
        head = blockIdx.x % p.kv_heads;
        row = y;
        // with the lengths where all CTAs have a row; where many have none, they go without it
        uint64_t total = 0, before = 0;
        if (W == 32) total = p.prefix[p.seqs], before = p.prefix[b];
        s = attn_seq(p, b, false);
        const ARShape sh = ar_shape<DP>(p, s);
        if (sh.tiles == 0 || row >= s.ql * p.group) return;
        if (W != 32) total = p.prefix[p.seqs], before = p.prefix[b];
        const uint64_t even = quotient(total + p.workers - 1, p.workers);
        const uint64_t per = even > p.least ? even : p.least;
        const uint64_t first = before + AR_UNIT_COST +
                               static_cast<uint64_t>(head * sh.tiles + row / AR_ROWS) * (sh.steps + AR_UNIT_COST);
        w0 = quotient(first, per);
        n = static_cast<uint32_t>(quotient(first + sh.steps - 1, per) - w0) + 1;
        if (n == 1) return; // written by its one warp
    }
    const uint32_t t = row / p.group, g = row % p.group, in = row % AR_ROWS;
    float acc[V] = {}, m = -INFINITY, l = 0.0f;
    for (uint32_t f0 = warp; f0 < n; f0 += F * W) {
        float2 ml[F];
        float v[F][V];
#pragma unroll
        for (uint32_t x = 0; x < F; ++x) {
            const uint32_t f = f0 + x * W;
            ml[x] = make_float2(-INFINITY, 0.0f);
            if (f < n) {
                const uint64_t slot = ((w0 + f) * 2 + (f == 0 ? 1 : 0)) * AR_ROWS + in;
                ml[x] = p.part_ml[slot];
#pragma unroll
                for (int i = 0; i < V; ++i) v[x][i] = p.part[slot * DP + col0 + lane * V + i];
            }
        }
#pragma unroll
        for (uint32_t x = 0; x < F; ++x) {
            if (f0 + x * W >= n) break;
            // a fragment without a largest exponent weighs nothing, but is added: if its scores
            // were NaN so are its sums, and times zero they stay that
            const float to = fmaxf(m, ml[x].x);
            const float fa = m == -INFINITY ? 0.0f : exp2_approx(m - to);
            const float fb = ml[x].x == -INFINITY ? 0.0f : exp2_approx(ml[x].x - to);
            m = to;
            l = l * fa + ml[x].y * fb;
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] = acc[i] * fa + v[x][i] * fb;
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) s_o[warp][lane * V + i] = acc[i];
    if (lane == 0) {
        s_m[warp] = m;
        s_l[warp] = l;
    }
    __syncthreads();
    const uint32_t in_part = threadIdx.x * 2, col = col0 + in_part;
    if (in_part >= DP / C || col >= p.dim) return;
    float top = -INFINITY, sum = 0.0f, a0 = 0.0f, a1 = 0.0f;
#pragma unroll
    for (uint32_t w = 0; w < W; ++w) top = fmaxf(top, s_m[w]);
#pragma unroll
    for (uint32_t w = 0; w < W; ++w) {
        const float f = s_m[w] == -INFINITY ? 0.0f : exp2_approx(s_m[w] - top);
        sum += s_l[w] * f;
        a0 += s_o[w][in_part] * f;
        a1 += s_o[w][in_part + 1] * f;
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const uint64_t h = head * p.group + g, token = static_cast<uint64_t>(s.q0) + t;
    *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(p.out) + token * p.ot + h * p.oh + col) =
        pack_pair<BF16>(a0 * inv, a1 * inv);
    if (p.lse && col == 0)
        p.lse[token * p.heads + h] = sum == 0.0f ? -INFINITY : top * 0.6931471805599453f + logf(sum);
}

} // namespace fmb
