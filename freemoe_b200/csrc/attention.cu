// attention.cu -- attention of new tokens over a paged cache: argument checks,
// workspace and launches.  Sequences with few rows go to the kernel that is
// limited by reading the cache (attention_rows.cuh), the others to the one on
// the tensor cores (attention_prompt.cuh); each finds its sequences from the
// lengths on the device, what the bounds rule out is not launched, and where
// both have work they are parts of one grid.
#include <cudaTypedefs.h>

#include <cmath>
#include <mutex>
#include <string>
#include <utility>

#include "attention_prompt.cuh"
#include "launch.cuh"

namespace fmb {
namespace {

inline uint64_t a256(uint64_t v) { return (v + 255) & ~uint64_t(255); }

// Steps a warp up to which the cluster form is taken: beyond, a wave of all SMs and the
// kernel that joins the fragments cost less than the SMs that the clusters leave idle.
constexpr uint32_t CLUSTER_STEPS = 16;

// Keys up to which a unit is one warp's.  Measured against ranges cut evenly, heads of 128:
// 160 units of 128 keys 9.8 against 13 us, of up to 256 keys 15.8 against 13 to 16, of up to
// 400 keys 22 against 14; 1024 units of up to 256 keys 20 against 26.
constexpr uint32_t UNIT_KEYS = 256;

// Rows (tokens x group) up to which a sequence is the rows kernel's: one tile of 16, or
// two, which read the cache twice (the second time from L2), where all of the batch's keys
// and values are few (by their bound, max_kv_len each).  Measured, 32 rows a sequence and
// key head, 8 key heads of 128, ragged lengths up to 4096 keys: 16 sequences 54 us there
// against 60 on the prompt kernel, 64 sequences 181 against 136.
constexpr uint32_t MOST_ROWS = 2 * AR_ROWS;
constexpr uint64_t TWICE_BYTES = 256u << 20;

// The prompt kernel's work is dealt out by blocks where whole items would leave
// CTAs idle: with fewer than DEAL_ITEMS items a CTA, or one a CTA where one
// prompt without context brings its own small items.  Items of up to WHOLE_BLOCKS
// blocks are not worth the fragments and the kernel that joins them.
constexpr uint32_t DEAL_ITEMS = 6, WHOLE_BLOCKS = 10;

struct AttnPlan {
    uint32_t dp, workers, group;
    uint32_t row_limit;
    bool rows, prompt;       // which kernels have work
    uint32_t cluster;        // CTAs a unit of the cluster form of the rows kernel; 0: the other form
    bool units;              // a warp a unit
    uint32_t tiles;          // row tiles of a unit's sequence and head, at most
    bool deal;               // prompt kernel: blocks are dealt out, not items
    uint32_t pairs, ctas;    // its pairs of tiles (a bound), and its grid
    uint64_t prefix, part, part_ml, tail_rows, ppart, ppart_ml, tail, total; // workspace offsets
};

// Keys that `rows` packed rows of a sequence see together, at most.
uint64_t keys_seen(const fmcuda_paged_attention_args &a, uint32_t rows) {
    const uint64_t seen = static_cast<uint64_t>(a.window) + rows / (a.heads / a.kv_heads) + 1;
    return a.window && seen < a.max_kv_len ? seen : a.max_kv_len;
}

AttnPlan attn_plan(const fmcuda_paged_attention_args &a) {
    AttnPlan n{};
    n.dp = a.head_dim <= 64 ? 64 : 128;
    n.group = a.heads / a.kv_heads;
    const uint32_t sms = static_cast<uint32_t>(device_sm_count());
    n.workers = sms * AR_WARPS;
    const uint64_t all = static_cast<uint64_t>(a.tokens) * n.group;
    const uint64_t bytes = keys_seen(a, MOST_ROWS) * a.seqs * a.kv_heads * a.head_dim * 4;
    n.row_limit = bytes <= TWICE_BYTES ? MOST_ROWS : AR_ROWS;
    n.prompt = static_cast<uint64_t>(a.max_q_len) * n.group > n.row_limit;
    // a sequence has at least tokens - (seqs - 1) * max_q_len rows, where that bound can be
    // true; without the rows kernel the other one takes sequences of any length
    const uint64_t others = static_cast<uint64_t>(a.seqs - 1) * a.max_q_len;
    n.rows = all <= others * n.group + n.row_limit || a.tokens > others + a.max_q_len;
    uint64_t o = 0;
    auto take = [&](uint64_t bytes) {
        const uint64_t at = o;
        o += a256(bytes);
        return at;
    };
    const uint64_t most_rows = static_cast<uint64_t>(a.max_q_len) * n.group;
    n.tiles = static_cast<uint32_t>((most_rows < n.row_limit ? most_rows + AR_ROWS - 1 : n.row_limit) / AR_ROWS);
    const uint64_t keys = keys_seen(a, MOST_ROWS);
    const uint64_t units = static_cast<uint64_t>(a.seqs) * a.kv_heads * n.tiles;
    if (n.rows && units && units <= sms) {
        // the largest cluster that one wave holds and that has a step for each warp
        const uint64_t steps = keys / ar_keys(static_cast<int>(n.dp)) + 1;
        // (a grid that takes chunks too has none: ranges and their join, a chunk of 150 behind 1500
        // keys beside 3 sequences 43 us, against 38 for clusters of 4 in a launch beside the chunk's)
        uint32_t c = n.prompt ? 1 : AR_MAX_CLUSTER;
        while (c > 1 && (units * c > sms || steps < c * AR_WARPS)) c /= 2;
        if (steps <= static_cast<uint64_t>(c) * AR_WARPS * CLUSTER_STEPS) n.cluster = c;
    }
    n.units = n.rows && !n.cluster && keys <= UNIT_KEYS;
    if (n.rows && !n.cluster && !n.units) {
        n.prefix = take((static_cast<uint64_t>(a.seqs) + 1) * 8);
        n.part = take(static_cast<uint64_t>(n.workers) * 2 * AR_ROWS * n.dp * 4);
        n.part_ml = take(static_cast<uint64_t>(n.workers) * 2 * AR_ROWS * 8);
        n.tail_rows = take(static_cast<uint64_t>(n.workers) * 16);
    }
    if (n.prompt) {
        const uint64_t big = all / ((n.rows ? n.row_limit : 0) + 1);
        n.pairs = static_cast<uint32_t>(all / AP_PAIR + (big < a.seqs ? big : a.seqs));
        const uint64_t items = static_cast<uint64_t>(n.pairs) * a.kv_heads;
        const bool prompt = a.seqs == 1 && a.causal && !a.window && a.max_q_len == a.max_kv_len;
        n.deal = items < static_cast<uint64_t>(sms) * (prompt ? 1 : DEAL_ITEMS) && n.pairs <= AP_MAX_PAIRS &&
                 keys_seen(a, AP_PAIR) > AP_KEYS * WHOLE_BLOCKS;
        n.ctas = !n.deal && items < sms ? static_cast<uint32_t>(items) : sms;
        if (n.deal) {
            n.ppart = take(static_cast<uint64_t>(n.ctas) * 2 * AP_PAIR * n.dp * 4);
            n.ppart_ml = take(static_cast<uint64_t>(n.ctas) * 2 * AP_PAIR * 8);
            n.tail = take(static_cast<uint64_t>(n.ctas) * 16);
        }
    }
    n.total = o;
    return n;
}

int check_attention(const fmcuda_paged_attention_args *a) {
    if (!a) return set_error(FM_STATUS_INVALID_ARGUMENT, "null attention arguments");
    if (a->dtype != FM_X_BF16 && a->dtype != FM_X_F16)
        return set_error(FM_STATUS_INVALID_ARGUMENT, "attention takes bfloat16 or float16");
    if (a->head_dim == 0 || a->head_dim % 8 || a->head_dim > 128)
        return set_error(FM_STATUS_SHAPE_MISMATCH, "head_dim must be a multiple of 8, at most 128");
    if (a->kv_heads == 0 || a->heads == 0 || a->heads % a->kv_heads || a->heads > 65535)
        return set_error(FM_STATUS_SHAPE_MISMATCH, "heads must be a multiple of kv_heads, at most 65535");
    if (a->page_size == 0 || a->page_size % 8 || a->page_size > (1u << 20))
        return set_error(FM_STATUS_SHAPE_MISMATCH, "page_size must be a multiple of 8, at most 2^20");
    if (a->max_kv_len > 0x7FFFFFFFu - 256 || a->tokens > 0x7FFFFFFFu || a->max_q_len > a->tokens ||
        a->n_pages > 0x7FFFFFFFu)
        return set_error(FM_STATUS_SHAPE_MISMATCH, "attention lengths out of range");
    if (static_cast<uint64_t>(a->tokens) * a->heads > 0x7FFFFFFFu ||
        static_cast<uint64_t>(a->seqs) * a->kv_heads > 0x7FFFFFFFu)
        return set_error(FM_STATUS_SHAPE_MISMATCH, "too many rows in a call");
    if (a->window && !a->causal) return set_error(FM_STATUS_INVALID_ARGUMENT, "a window needs causal attention");
    if (!(a->scale > 0.0f) || !std::isfinite(a->scale))
        return set_error(FM_STATUS_INVALID_ARGUMENT, "attention scale must be positive and finite");
    if (a->page_table_stride < static_cast<int64_t>((a->max_kv_len + a->page_size - 1) / a->page_size))
        return set_error(FM_STATUS_SHAPE_MISMATCH, "page table is shorter than max_kv_len");
    const int64_t strides[] = {a->q_token_stride,    a->q_head_stride,     a->out_token_stride, a->out_head_stride,
                               a->cache_page_stride, a->cache_head_stride, a->cache_row_stride};
    for (int64_t s : strides)
        if (s < 0 || s % 8) return set_error(FM_STATUS_SHAPE_MISMATCH, "attention strides must be multiples of 8");
    return FM_STATUS_OK;
}

// The cache as boxes of 64 values x box_rows rows of one head of one page, the
// dimensions in the order of their strides (`heads_first`: a page's heads lie
// inside its rows).
int make_cache_map(CUtensorMap *map, const fmcuda_paged_attention_args &a, const void *base, uint32_t box_rows,
                   bool heads_first) {
    static std::once_flag once;
    static PFN_cuTensorMapEncodeTiled_v12000 enc = nullptr;
    std::call_once(once, [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            enc = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
        else
            (void)cudaGetLastError();
    });
    if (!enc) return set_error(FM_STATUS_INTERNAL_ERROR, "cuTensorMapEncodeTiled is unavailable");
    cuuint64_t dims[4] = {a.head_dim, a.page_size, a.kv_heads, a.n_pages ? a.n_pages : 1u};
    cuuint64_t strides[3] = {static_cast<cuuint64_t>(a.cache_row_stride) * 2,
                             static_cast<cuuint64_t>(a.cache_head_stride) * 2,
                             static_cast<cuuint64_t>(a.cache_page_stride) * 2};
    cuuint32_t box[4] = {64, box_rows, 1, 1}, step[4] = {1, 1, 1, 1};
    if (heads_first) {
        std::swap(dims[1], dims[2]);
        std::swap(strides[0], strides[1]);
        std::swap(box[1], box[2]);
    }
    const CUresult r =
        enc(map, a.dtype == FM_X_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
            const_cast<void *>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return set_error(FM_STATUS_INVALID_ARGUMENT,
                         "the cache's strides do not make a tensor map (" + std::to_string(r) + ")");
    return FM_STATUS_OK;
}

template <int DP, bool BF16>
int launch_attention(const fmcuda_paged_attention_args &a, const AttnPlan &n, const AttnParams &p, uint8_t *ws,
                     cudaStream_t s) {
    int rc = FM_STATUS_OK;
    // sequences of few rows: a cluster a unit; a warp a unit, one a CTA until there is one on every
    // SM; or ranges
    const uint64_t row_units = static_cast<uint64_t>(p.seqs) * p.kv_heads * n.tiles, sms = device_sm_count();
    const uint32_t unit_warps = row_units < sms * AR_WARPS ? static_cast<uint32_t>((row_units + sms - 1) / sms) : AR_WARPS;
    const uint32_t rows_ctas = n.cluster ? static_cast<uint32_t>(row_units) * n.cluster
                               : n.units ? static_cast<uint32_t>((row_units + unit_warps - 1) / unit_warps)
                                         : p.workers / AR_WARPS;
    APParams pp{};
    if (n.prompt) {
        pp.a = p;
        pp.box_rows = a.page_size & (~a.page_size + 1u); // its lowest set bit
        if (pp.box_rows > AP_KEYS) pp.box_rows = AP_KEYS;
        pp.heads_first = a.cache_head_stride < a.cache_row_stride;
        pp.wide = a.head_dim % 16 == 0 && a.out_token_stride % 16 == 0 && a.out_head_stride % 16 == 0 &&
                  reinterpret_cast<uintptr_t>(a.out) % 32 == 0;
        pp.deal = n.deal;
        pp.max_pairs = n.pairs;
        pp.part = reinterpret_cast<float *>(ws + n.ppart);
        pp.part_ml = reinterpret_cast<float2 *>(ws + n.ppart_ml);
        pp.tail = reinterpret_cast<int4 *>(ws + n.tail);
        pp.ctas = n.ctas;
        pp.rows_form = n.cluster ? AR_CLUSTER : n.units ? AR_UNIT : AR_RANGES;
        pp.rows_tiles = n.tiles;
        pp.rows_warps = unit_warps;
        CUtensorMap map_k, map_v;
        rc = make_cache_map(&map_k, a, a.k_cache, pp.box_rows, pp.heads_first);
        if (!rc) rc = make_cache_map(&map_v, a, a.v_cache, pp.box_rows, pp.heads_first);
        if (!rc && n.rows)
            rc = launch("attn_beside_kernel", attn_beside_kernel<DP, BF16>,
                        {dim3(n.ctas + rows_ctas), AP_THREADS, AP_BESIDE_SMEM<DP>, 1}, s, map_k, map_v, pp);
        else if (!rc)
            rc = launch("attn_prompt_kernel", attn_prompt_kernel<DP, BF16>,
                        {dim3(n.ctas), AP_THREADS, APrompt<DP>::SMEM, 1}, s, map_k, map_v, pp);
    } else if (n.cluster) {
        rc = launch("attn_cluster_kernel", attn_cluster_kernel<DP, BF16>,
                    {dim3(rows_ctas), AR_THREADS, ARows<DP>::SMEM, n.cluster}, s, p, n.tiles);
    } else if (n.units) {
        rc = launch("attn_unit_kernel", attn_unit_kernel<DP, BF16>,
                    {dim3(rows_ctas), unit_warps * 32, ARows<DP>::RINGS / AR_WARPS * unit_warps, 1}, s, p, n.tiles);
    } else {
        rc = launch("attn_rows_kernel", attn_rows_kernel<DP, BF16>, {dim3(rows_ctas), AR_THREADS, ARows<DP>::SMEM, 1}, s,
                    p);
    }
    if (!rc && n.prompt && n.deal)
        rc = launch("attn_join_kernel", attn_join_kernel<DP, BF16>, {dim3(n.ctas, AJ_SLICES), 256, 0, 1}, s, pp);
    if (rc || !n.rows || n.cluster || n.units) return rc;
    const uint64_t most = static_cast<uint64_t>(a.max_q_len) * n.group, units = static_cast<uint64_t>(p.seqs) * p.kv_heads;
    const uint32_t rows = most < n.row_limit ? static_cast<uint32_t>(most) : n.row_limit;
    // few units are cut into many fragments each; of many units, few are cut
    if (units * 16 <= p.workers) {
        const dim3 whole(static_cast<uint32_t>(units), rows), parts(static_cast<uint32_t>(units), rows * 2);
        if (units * rows * 2 <= static_cast<uint64_t>(device_sm_count())) // one such CTA an SM
            return launch("attn_combine_kernel", attn_combine_kernel<DP, BF16, 32, 5, 2>, {parts, 32 * 32, 0, 1}, s, p, false);
        return launch("attn_combine_kernel", attn_combine_kernel<DP, BF16, 32, 5, 1>, {whole, 32 * 32, 0, 1}, s, p, false);
    }
    const bool by_worker = units * n.tiles > p.workers;
    const dim3 grid = by_worker ? dim3(p.workers, rows < AR_ROWS ? rows : AR_ROWS) : dim3(static_cast<uint32_t>(units), rows);
    return launch("attn_combine_kernel", attn_combine_kernel<DP, BF16, 4, 2, 1>, {grid, 4 * 32, 0, 1}, s, p, by_worker);
}

} // namespace
} // namespace fmb

using namespace fmb;

extern "C" int fmcuda_paged_attention_workspace_bytes(const fmcuda_paged_attention_args *args, uint64_t *bytes) {
    if (!bytes) return set_error(FM_STATUS_INVALID_ARGUMENT, "null workspace size");
    const int rc = check_attention(args);
    if (rc) return rc;
    *bytes = args->seqs ? attn_plan(*args).total : 0;
    return FM_STATUS_OK;
}

extern "C" int fmcuda_paged_attention(const fmcuda_paged_attention_args *a, void *workspace, uint64_t workspace_bytes,
                                      void *stream) {
    int rc = check_attention(a);
    if (rc) return rc;
    if (a->seqs == 0 || a->tokens == 0 || a->max_q_len == 0) return FM_STATUS_OK;
    if (!a->q || !a->k_cache || !a->v_cache || !a->out || !a->page_table || !a->q_start || !a->kv_len)
        return set_error(FM_STATUS_INVALID_ARGUMENT, "null attention buffer");
    const void *aligned[] = {a->q, a->k_cache, a->v_cache, a->out};
    for (const void *x : aligned)
        if (reinterpret_cast<uintptr_t>(x) % 16)
            return set_error(FM_STATUS_INVALID_ARGUMENT, "attention buffers must be 16-byte aligned");
    const void *words[] = {a->page_table, a->q_start, a->kv_len, a->lse};
    for (const void *x : words)
        if (reinterpret_cast<uintptr_t>(x) % 4)
            return set_error(FM_STATUS_INVALID_ARGUMENT, "lengths, pages and lse must be aligned to their values");
    const AttnPlan n = attn_plan(*a);
    if ((n.total && !workspace) || workspace_bytes < n.total || reinterpret_cast<uintptr_t>(workspace) % 256)
        return set_error(FM_STATUS_INVALID_ARGUMENT, "attention workspace is too small or not 256-byte aligned");
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    AttnParams p{};
    p.q = a->q;
    p.kc = a->k_cache;
    p.vc = a->v_cache;
    p.out = a->out;
    p.lse = a->lse;
    p.table = a->page_table;
    p.q_start = a->q_start;
    p.kv_len = a->kv_len;
    p.qt = a->q_token_stride;
    p.qh = a->q_head_stride;
    p.ot = a->out_token_stride;
    p.oh = a->out_head_stride;
    p.cp = a->cache_page_stride;
    p.ch = a->cache_head_stride;
    p.cr = a->cache_row_stride;
    p.tb = a->page_table_stride;
    p.seqs = a->seqs;
    p.tokens = a->tokens;
    p.heads = a->heads;
    p.kv_heads = a->kv_heads;
    p.group = a->heads / a->kv_heads;
    p.dim = a->head_dim;
    p.n_pages = a->n_pages;
    p.page_size = a->page_size;
    p.max_q = a->max_q_len;
    p.max_kv = a->max_kv_len;
    p.window = a->window;
    p.causal = a->causal;
    p.scale = a->scale;
    p.scale_log2 = a->scale * 1.4426950408889634f;
    p.status = device_status_word();
    p.prefix = reinterpret_cast<uint64_t *>(ws + n.prefix);
    p.part = reinterpret_cast<float *>(ws + n.part);
    p.part_ml = reinterpret_cast<float2 *>(ws + n.part_ml);
    p.tail_rows = reinterpret_cast<int4 *>(ws + n.tail_rows);
    p.workers = n.workers;
    p.least = 4;
    p.row_limit = n.rows ? n.row_limit : 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool bf = a->dtype == FM_X_BF16;
    if (n.dp == 64)
        return bf ? launch_attention<64, true>(*a, n, p, ws, s) : launch_attention<64, false>(*a, n, p, ws, s);
    return bf ? launch_attention<128, true>(*a, n, p, ws, s) : launch_attention<128, false>(*a, n, p, ws, s);
}
