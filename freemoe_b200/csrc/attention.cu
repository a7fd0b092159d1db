// attention.cu -- attention of new tokens over a paged cache: argument checks,
// workspace and launches.  Sequences with few rows go to the kernel that is
// limited by reading the cache (attention_rows.cuh), the others to the one on
// the tensor cores (attention_prompt.cuh); each finds its sequences from the
// lengths on the device, what the bounds rule out is not launched, and where
// both have work they are parts of one grid.
#include <cmath>
#include <string>

#include "attention_launch.cuh"

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

// Keys that `rows` packed rows of a sequence see together, at most.
uint64_t keys_seen(const fmcuda_paged_attention_args &a, uint32_t sinks, uint32_t rows) {
    const uint64_t seen = static_cast<uint64_t>(a.window) + sinks + rows / (a.heads / a.kv_heads) + 1;
    return a.window && seen < a.max_kv_len ? seen : a.max_kv_len;
}

AttnPlan attn_plan(const fmcuda_paged_attention_args &a, uint32_t sinks) {
    AttnPlan n{};
    n.dp = a.head_dim <= 64 ? 64 : 128;
    n.group = a.heads / a.kv_heads;
    const uint32_t sms = static_cast<uint32_t>(device_sm_count());
    n.workers = sms * AR_WARPS;
    const uint64_t all = static_cast<uint64_t>(a.tokens) * n.group;
    const uint64_t bytes = keys_seen(a, sinks, MOST_ROWS) * a.seqs * a.kv_heads * a.head_dim * 4;
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
    const uint64_t keys = keys_seen(a, sinks, MOST_ROWS);
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
                 keys_seen(a, sinks, AP_PAIR) > AP_KEYS * WHOLE_BLOCKS;
        n.ctas = !n.deal && items < sms ? static_cast<uint32_t>(items) : sms;
        // with first keys single tiles may be items, on the SMs that sequences of few rows leave: a CTA
        // a unit, or all (39 decoding sequences beside a chunk of 56 items 38 us, with 112 of single tiles 47)
        const uint64_t beside = !n.rows ? 0 : n.cluster || n.units ? static_cast<uint64_t>(a.seqs) * a.kv_heads : sms;
        if (sinks && !n.deal && beside < sms) {
            n.singles = static_cast<uint32_t>(items * 2 < sms - beside ? items * 2 : sms - beside);
            n.ctas = n.ctas > n.singles ? n.ctas : n.singles;
        }
        if (n.deal) {
            n.ppart = take(static_cast<uint64_t>(n.ctas) * 2 * AP_PAIR * n.dp * 4);
            n.ppart_ml = take(static_cast<uint64_t>(n.ctas) * 2 * AP_PAIR * 8);
            n.tail = take(static_cast<uint64_t>(n.ctas) * 16);
        }
    }
    n.total = o;
    return n;
}

int check_attention(const fmcuda_paged_attention_args *a, uint32_t sinks) {
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
    if (sinks && !a->window) return set_error(FM_STATUS_INVALID_ARGUMENT, "first keys stay visible behind a window");
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

} // namespace
} // namespace fmb

using namespace fmb;

extern "C" int fmcuda_paged_attention_sinks_workspace_bytes(const fmcuda_paged_attention_args *args, uint32_t sinks,
                                                            uint64_t *bytes) {
    if (!bytes) return set_error(FM_STATUS_INVALID_ARGUMENT, "null workspace size");
    const int rc = check_attention(args, sinks);
    if (rc) return rc;
    *bytes = args->seqs ? attn_plan(*args, sinks).total : 0;
    return FM_STATUS_OK;
}

extern "C" int fmcuda_paged_attention_workspace_bytes(const fmcuda_paged_attention_args *args, uint64_t *bytes) {
    return fmcuda_paged_attention_sinks_workspace_bytes(args, 0, bytes);
}

extern "C" int fmcuda_paged_attention_sinks(const fmcuda_paged_attention_args *a, uint32_t sinks, void *workspace,
                                            uint64_t workspace_bytes, void *stream) {
    const int rc = check_attention(a, sinks);
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
    const AttnPlan n = attn_plan(*a, sinks);
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
    p.sinks = sinks < a->max_kv_len ? sinks : a->max_kv_len; // its roundings stay in 32 bits
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
    return sinks ? launch_attention_sinks(*a, n, p, ws, s) : launch_attention_of<false>(*a, n, p, ws, s);
}

extern "C" int fmcuda_paged_attention(const fmcuda_paged_attention_args *a, void *workspace, uint64_t workspace_bytes,
                                      void *stream) {
    return fmcuda_paged_attention_sinks(a, 0, workspace, workspace_bytes, stream);
}
