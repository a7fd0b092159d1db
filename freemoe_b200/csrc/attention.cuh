// attention.cuh -- what the kernels of attention over a paged cache share: the
// arguments, the shape of a sequence's work, and the layout of partial results.
#pragma once

#include "common.cuh"
#include "launch.cuh"
#include "ptx.cuh"

namespace fmb {

struct AttnParams {
    const void *q, *kc, *vc;
    void *out;
    float *lse;
    const int32_t *table, *q_start, *kv_len;
    int64_t qt, qh, ot, oh, cp, ch, cr, tb;
    uint32_t seqs, tokens, heads, kv_heads, group, dim;
    uint32_t n_pages, page_size;
    uint32_t max_q, max_kv;
    uint32_t window; // 0: none
    int32_t causal;
    float scale, scale_log2; // scale, and scale * log2(e)
    int *status;
    uint64_t *prefix; // [seqs + 1]: steps of the rows kernel before each sequence
    float *part;      // partial sums
    float2 *part_ml;  // their (largest exponent in log2, sum)
    int4 *tail_rows;         // [workers]: the unit that begins in a warp's range and is cut: sequence (or -1), tile, fragments
    uint32_t workers, least; // rows kernel: warps, and the least work of a warp, in steps
    uint32_t row_limit;      // rows x group up to which a sequence is the rows kernel's
};

// One sequence: first row and number of rows, keys, and the first key that any row sees.
struct AttnSeq {
    uint32_t q0, ql, kl, lo;
};

__device__ __forceinline__ AttnSeq attn_seq(const AttnParams &p, uint32_t b, bool report) {
    AttnSeq s;
    const int32_t q0 = __ldg(p.q_start + b), q1 = __ldg(p.q_start + b + 1), kl = __ldg(p.kv_len + b);
    bool bad = false;
    s.q0 = static_cast<uint32_t>(q0);
    s.ql = static_cast<uint32_t>(q1 - q0);
    if (q0 < 0 || q1 < q0 || static_cast<uint32_t>(q1) > p.tokens) {
        bad = true;
        s.q0 = s.ql = 0;
    }
    if (s.ql > p.max_q) {
        bad = true;
        s.ql = 0;
    }
    s.kl = static_cast<uint32_t>(kl);
    if (kl < 0 || s.kl > p.max_kv) {
        bad = true;
        s.kl = 0;
    }
    if (bad && report) raise_device_status(p.status, FM_STATUS_INVALID_ARGUMENT);
    s.lo = 0;
    if (p.window) {
        const int64_t lo = static_cast<int64_t>(s.kl) - s.ql - p.window + 1;
        s.lo = lo > 0 ? static_cast<uint32_t>(lo) : 0;
    }
    return s;
}

// A 64-bit quotient by a 32-bit division where that does (it takes a fifth of the time, and the
// first thing that a kernel does is to find its work).
__device__ __forceinline__ uint64_t quotient(uint64_t a, uint64_t b) {
    return (a | b) >> 32 ? a / b : static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}

template <bool BF16> __device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
    uint32_t r;
    if constexpr (BF16)
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
    else
        asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

} // namespace fmb
