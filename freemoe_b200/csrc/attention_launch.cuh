// attention_launch.cuh -- the launches of attention over a paged cache, for a plan that
// the entry point made; instantiated without and with first keys that stay visible
// (attention.cu, attention_sinks.cu).
#pragma once

#include <cudaTypedefs.h>

#include <mutex>
#include <string>
#include <utility>

#include "attention_prompt.cuh"
#include "launch.cuh"

namespace fmb {

struct AttnPlan {
    uint32_t dp, workers, group;
    uint32_t row_limit;
    bool rows, prompt;       // which kernels have work
    uint32_t cluster;        // CTAs a unit of the cluster form of the rows kernel; 0: the other form
    bool units;              // a warp a unit
    uint32_t tiles;          // row tiles of a unit's sequence and head, at most
    bool deal;               // prompt kernel: blocks are dealt out, not items
    uint32_t pairs, ctas;    // its pairs of tiles (a bound), and its grid
    uint32_t singles;        // CTAs that may take single tiles
    uint64_t prefix, part, part_ml, tail_rows, ppart, ppart_ml, tail, total; // workspace offsets
};

// The cache as boxes of 64 values x box_rows rows of one head of one page, the
// dimensions in the order of their strides (`heads_first`: a page's heads lie
// inside its rows).
inline int make_cache_map(CUtensorMap *map, const fmcuda_paged_attention_args &a, const void *base, uint32_t box_rows,
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

template <int DP, bool BF16, bool SINKS>
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
        pp.singles = n.singles;
        pp.rows_form = n.cluster ? AR_CLUSTER : n.units ? AR_UNIT : AR_RANGES;
        pp.rows_tiles = n.tiles;
        pp.rows_warps = unit_warps;
        CUtensorMap map_k, map_v;
        rc = make_cache_map(&map_k, a, a.k_cache, pp.box_rows, pp.heads_first);
        if (!rc) rc = make_cache_map(&map_v, a, a.v_cache, pp.box_rows, pp.heads_first);
        if (!rc && n.rows)
            rc = launch("attn_beside_kernel", attn_beside_kernel<DP, BF16, SINKS>,
                        {dim3(n.ctas + rows_ctas), AP_THREADS, AP_BESIDE_SMEM<DP>, 1, AP_BESIDE_SMEM<DP>}, s, map_k,
                        map_v, pp);
        else if (!rc)
            rc = launch("attn_prompt_kernel", attn_prompt_kernel<DP, BF16, SINKS>,
                        {dim3(n.ctas), AP_THREADS, APrompt<DP>::SMEM, 1, APrompt<DP>::SMEM}, s, map_k, map_v, pp);
    } else if (n.cluster) {
        rc = launch("attn_cluster_kernel", attn_cluster_kernel<DP, BF16, SINKS>,
                    {dim3(rows_ctas), AR_THREADS, ARows<DP>::SMEM, n.cluster, ARows<DP>::SMEM}, s, p, n.tiles);
    } else if (n.units) {
        rc = launch("attn_unit_kernel", attn_unit_kernel<DP, BF16, SINKS>,
                    {dim3(rows_ctas), unit_warps * 32, ARows<DP>::RINGS / AR_WARPS * unit_warps, 1, ARows<DP>::RINGS}, s,
                    p, n.tiles);
    } else {
        rc = launch("attn_rows_kernel", attn_rows_kernel<DP, BF16, SINKS>,
                    {dim3(rows_ctas), AR_THREADS, ARows<DP>::SMEM, 1, ARows<DP>::SMEM}, s, p);
    }
    if (!rc && n.prompt && n.deal)
        rc = launch("attn_join_kernel", attn_join_kernel<DP, BF16>, {dim3(n.ctas, AJ_SLICES), 256, 0, 1, 0}, s, pp);
    if (rc || !n.rows || n.cluster || n.units) return rc;
    const uint64_t most = static_cast<uint64_t>(a.max_q_len) * n.group, units = static_cast<uint64_t>(p.seqs) * p.kv_heads;
    const uint32_t rows = most < n.row_limit ? static_cast<uint32_t>(most) : n.row_limit;
    // few units are cut into many fragments each; of many units, few are cut
    if (units * 16 <= p.workers) {
        const dim3 whole(static_cast<uint32_t>(units), rows), parts(static_cast<uint32_t>(units), rows * 2);
        if (units * rows * 2 <= static_cast<uint64_t>(device_sm_count())) // one such CTA an SM
            return launch("attn_combine_kernel", attn_combine_kernel<DP, BF16, SINKS, 32, 5, 2>, {parts, 32 * 32, 0, 1, 0}, s, p, false);
        return launch("attn_combine_kernel", attn_combine_kernel<DP, BF16, SINKS, 32, 5, 1>, {whole, 32 * 32, 0, 1, 0}, s, p, false);
    }
    const bool by_worker = units * n.tiles > p.workers;
    const dim3 grid = by_worker ? dim3(p.workers, rows < AR_ROWS ? rows : AR_ROWS) : dim3(static_cast<uint32_t>(units), rows);
    return launch("attn_combine_kernel", attn_combine_kernel<DP, BF16, SINKS, 4, 2, 1>, {grid, 4 * 32, 0, 1, 0}, s, p, by_worker);
}

// By the plan's padded head width and the arguments' type.
template <bool SINKS>
int launch_attention_of(const fmcuda_paged_attention_args &a, const AttnPlan &n, const AttnParams &p, uint8_t *ws,
                        cudaStream_t s) {
    const bool bf = a.dtype == FM_X_BF16;
    if (n.dp == 64)
        return bf ? launch_attention<64, true, SINKS>(a, n, p, ws, s) : launch_attention<64, false, SINKS>(a, n, p, ws, s);
    return bf ? launch_attention<128, true, SINKS>(a, n, p, ws, s) : launch_attention<128, false, SINKS>(a, n, p, ws, s);
}

int launch_attention_sinks(const fmcuda_paged_attention_args &a, const AttnPlan &n, const AttnParams &p, uint8_t *ws,
                           cudaStream_t s);

} // namespace fmb
