// attention.cu -- attention of new tokens over a paged cache: argument checks,
// workspace and launches.  Sequences with few rows go to the kernel that is
// limited by reading the cache (attention_rows.cuh), the others to the one on
// the tensor cores (attention_prompt.cuh); each kernel finds its sequences
// from the lengths on the device, and a kernel that the bounds rule out is not
// launched.
#include <cudaTypedefs.h>

#include <cmath>
#include <mutex>
#include <string>
#include <utility>

#include "attention_prompt.cuh"
#include "attention_rows.cuh"

namespace fmb {
namespace {

inline uint64_t a256(uint64_t v) { return (v + 255) & ~uint64_t(255); }

// Rows (tokens x group) up to which a sequence is the rows kernel's.
constexpr uint32_t ROW_LIMIT = 32;

struct AttnPlan {
    uint32_t dp, workers, group;
    bool rows, prompt;       // which kernels have work
    uint32_t pairs, splits;  // prompt kernel: bound on its tile pairs, parts of a pair
    uint64_t prefix, part, part_ml, ppart, ppart_ml, total; // workspace offsets
};

AttnPlan attn_plan(const fmcuda_paged_attention_args &a) {
    AttnPlan n{};
    n.dp = a.head_dim <= 64 ? 64 : 128;
    n.group = a.heads / a.kv_heads;
    const uint32_t sms = static_cast<uint32_t>(device_sm_count());
    n.workers = sms * AR_WARPS;
    const uint64_t all = static_cast<uint64_t>(a.tokens) * n.group;
    n.prompt = static_cast<uint64_t>(a.max_q_len) * n.group > ROW_LIMIT;
    // a sequence has at least tokens - (seqs - 1) * max_q_len rows, where that bound can be
    // true; without the rows kernel the other one takes sequences of any length
    const uint64_t others = static_cast<uint64_t>(a.seqs - 1) * a.max_q_len;
    n.rows = all <= others * n.group + ROW_LIMIT || a.tokens > others + a.max_q_len;
    uint64_t o = 0;
    auto take = [&](uint64_t bytes) {
        const uint64_t at = o;
        o += a256(bytes);
        return at;
    };
    if (n.rows) {
        n.prefix = take((static_cast<uint64_t>(a.seqs) + 1) * 8);
        n.part = take(static_cast<uint64_t>(n.workers) * 2 * AR_ROWS * n.dp * 4);
        n.part_ml = take(static_cast<uint64_t>(n.workers) * 2 * AR_ROWS * 8);
    }
    n.splits = 1;
    if (n.prompt) {
        const uint64_t big = all / ((n.rows ? ROW_LIMIT : 0) + 1);
        n.pairs = static_cast<uint32_t>(all / AP_PAIR + (big < a.seqs ? big : a.seqs));
        // fewer pairs than SMs: split their keys until every SM has a part
        const uint64_t want = (all + AP_PAIR - 1) / AP_PAIR * a.kv_heads;
        const uint64_t most = a.max_kv_len / (AP_KEYS * AP_LEAST_BLOCKS);
        uint64_t splits = want < sms ? sms / want : 1;
        splits = splits < most ? splits : most;
        n.splits = splits < 1 ? 1 : static_cast<uint32_t>(splits);
        if (n.splits > 1) {
            const uint64_t slots = static_cast<uint64_t>(n.pairs) * a.kv_heads * n.splits * AP_PAIR;
            n.ppart = take(slots * n.dp * 4);
            n.ppart_ml = take(slots * 8);
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
    attn_combine_kernel<DP, BF16><<<dim3(p.seqs * p.kv_heads, rows), AC_THREADS, 0, s>>>(p);
    return check_launch("attn_combine_kernel");
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
int launch_prompt(const fmcuda_paged_attention_args &a, const AttnPlan &n, const AttnParams &ap, uint8_t *ws,
                  cudaStream_t s) {
    using L = APrompt<DP>;
    static bool ready[64] = {};
    auto kfn = attn_prompt_kernel<DP, BF16>;
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !ready[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM);
        if (e != cudaSuccess) return cuda_status(e, "attention shared memory");
        if (dev >= 0 && dev < 64) ready[dev] = true;
    }
    APParams p{};
    p.a = ap;
    p.box_rows = a.page_size & (~a.page_size + 1u); // its lowest set bit
    if (p.box_rows > AP_KEYS) p.box_rows = AP_KEYS;
    p.heads_first = a.cache_head_stride < a.cache_row_stride;
    p.splits = n.splits;
    p.part = reinterpret_cast<float *>(ws + n.ppart);
    p.part_ml = reinterpret_cast<float2 *>(ws + n.ppart_ml);
    CUtensorMap map_k, map_v;
    int rc = make_cache_map(&map_k, a, a.k_cache, p.box_rows, p.heads_first);
    if (!rc) rc = make_cache_map(&map_v, a, a.v_cache, p.box_rows, p.heads_first);
    if (rc) return rc;
    const uint64_t grid = static_cast<uint64_t>(n.pairs) * a.kv_heads * n.splits;
    if (grid > 0x7FFFFFFFu) return set_error(FM_STATUS_SHAPE_MISMATCH, "too many rows in a call");
    kfn<<<static_cast<uint32_t>(grid), AP_THREADS, L::SMEM, s>>>(map_k, map_v, p);
    rc = check_launch("attn_prompt_kernel");
    if (rc || n.splits == 1) return rc;
    const uint64_t rows = static_cast<uint64_t>(a.tokens) * a.heads;
    attn_join_kernel<DP, BF16><<<static_cast<uint32_t>((rows + 7) / 8), 256, 0, s>>>(p);
    return check_launch("attn_join_kernel");
}

template <int DP, bool BF16>
int launch_attention(const fmcuda_paged_attention_args &a, const AttnPlan &n, const AttnParams &p, uint8_t *ws,
                     cudaStream_t s) {
    int rc = FM_STATUS_OK;
    if (n.prompt) rc = launch_prompt<DP, BF16>(a, n, p, ws, s);
    if (rc || !n.rows) return rc;
    const uint64_t rows = static_cast<uint64_t>(a.max_q_len) * n.group;
    return launch_rows<DP, BF16>(p, rows < ROW_LIMIT ? static_cast<uint32_t>(rows) : ROW_LIMIT, s);
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
    p.workers = n.workers;
    p.least = 4;
    p.row_limit = n.rows ? ROW_LIMIT : 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool bf = a->dtype == FM_X_BF16;
    if (n.dp == 64)
        return bf ? launch_attention<64, true>(*a, n, p, ws, s) : launch_attention<64, false>(*a, n, p, ws, s);
    return bf ? launch_attention<128, true>(*a, n, p, ws, s) : launch_attention<128, false>(*a, n, p, ws, s);
}
