// attention.cu -- attention of new tokens over a paged cache: argument checks,
// workspace and launches (attention_rows.cuh).
#include <cmath>
#include <string>

#include "attention_rows.cuh"

namespace fmb {
namespace {

inline uint64_t a256(uint64_t v) { return (v + 255) & ~uint64_t(255); }

struct AttnPlan {
    uint32_t dp, workers;
    uint64_t prefix, part, part_ml, total; // workspace offsets
};

AttnPlan attn_plan(const fmcuda_paged_attention_args &a) {
    AttnPlan n{};
    n.dp = a.head_dim <= 64 ? 64 : 128;
    n.workers = static_cast<uint32_t>(device_sm_count()) * AR_WARPS;
    uint64_t o = 0;
    n.prefix = o;
    o += a256((static_cast<uint64_t>(a.seqs) + 1) * 8);
    n.part = o;
    o += a256(static_cast<uint64_t>(n.workers) * 2 * AR_ROWS * n.dp * 4);
    n.part_ml = o;
    o += a256(static_cast<uint64_t>(n.workers) * 2 * AR_ROWS * 8);
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
    if (a->window && !a->causal) return set_error(FM_STATUS_INVALID_ARGUMENT, "a window needs causal attention");
    if (!std::isfinite(a->scale)) return set_error(FM_STATUS_INVALID_ARGUMENT, "attention scale is not finite");
    if (a->page_table_stride < static_cast<int64_t>((a->max_kv_len + a->page_size - 1) / a->page_size))
        return set_error(FM_STATUS_SHAPE_MISMATCH, "page table is shorter than max_kv_len");
    const int64_t strides[] = {a->q_token_stride,    a->q_head_stride,     a->out_token_stride, a->out_head_stride,
                               a->cache_page_stride, a->cache_head_stride, a->cache_row_stride};
    for (int64_t s : strides)
        if (s < 0 || s % 8) return set_error(FM_STATUS_SHAPE_MISMATCH, "attention strides must be multiples of 8");
    return FM_STATUS_OK;
}

template <int DP, bool BF16> int launch_rows(const AttnParams &p, uint32_t rows, cudaStream_t s) {
    static bool ready[64] = {};
    auto kfn = attn_rows_kernel<DP, BF16>;
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !ready[dev]) {
        const cudaError_t e =
            cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, ARows<DP>::SMEM);
        if (e != cudaSuccess) return cuda_status(e, "attention shared memory");
        if (dev >= 0 && dev < 64) ready[dev] = true;
    }
    kfn<<<p.workers / AR_WARPS, AR_THREADS, ARows<DP>::SMEM, s>>>(p);
    int rc = check_launch("attn_rows_kernel");
    if (rc) return rc;
    attn_combine_kernel<DP, BF16><<<dim3(p.seqs * p.kv_heads, rows < 65535u ? rows : 65535u), AC_THREADS, 0, s>>>(p);
    return check_launch("attn_combine_kernel");
}

} // namespace
} // namespace fmb

using namespace fmb;

extern "C" int fmcuda_paged_attention_workspace_bytes(const fmcuda_paged_attention_args *args, uint64_t *bytes) {
    if (!bytes) return set_error(FM_STATUS_INVALID_ARGUMENT, "null workspace size");
    const int rc = check_attention(args);
    if (rc) return rc;
    *bytes = attn_plan(*args).total;
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
    const AttnPlan n = attn_plan(*a);
    if (!workspace || workspace_bytes < n.total || reinterpret_cast<uintptr_t>(workspace) % 256)
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
    p.workers = n.workers;
    p.least = 4;
    p.row_limit = 0xFFFFFFFFu;
    const uint64_t rows = static_cast<uint64_t>(a->max_q_len) * p.group;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool bf = a->dtype == FM_X_BF16;
    const uint32_t r = static_cast<uint32_t>(rows);
    if (n.dp == 64) return bf ? launch_rows<64, true>(p, r, s) : launch_rows<64, false>(p, r, s);
    return bf ? launch_rows<128, true>(p, r, s) : launch_rows<128, false>(p, r, s);
}
