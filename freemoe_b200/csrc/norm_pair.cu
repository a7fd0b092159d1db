// norm_pair.cu -- the norms around a block: the norm of the block's output, its gated
// and scaled addition to the residual stream, and the norm before the next block.
//
//   n = x w1 / sqrt(mean(x^2) + eps),  h = a r + s g n,  y = h w2 / sqrt(mean(h^2) + eps)
//
// The operator is one read of x and r (and of a gate of their shape) and one write of h
// and y.  The second mean is of h itself, not of the four sums that would give it in one
// pass over x and r: where the block's output cancels the stream those lose all their
// digits.
#include <cmath>
#include <string>

#include "launch.cuh"
#include "norm_rows.cuh"

namespace fmb {

namespace {

enum PairGate : int32_t { GATE_NONE, GATE_CHANNEL, GATE_TOKEN, GATE_FULL };

struct PairParams {
    const void *x, *w1, *gate, *res, *w2;
    void *y, *res_out;
    float *scales;
    int64_t xs, gs, rs, ys;
    int32_t xt, rt, wt, gt, yt;
    PairGate gate_kind;
    uint32_t tokens, d;
    float scale, res_scale, eps;
};

// h of chunk c: `by` is the factor of the row (its first norm, the scale, its gate).
template <int VEC>
__device__ __forceinline__ void pair_h(const PairParams &p, uint64_t row, uint32_t c, float by, float (&h)[8]) {
    float v[8];
    load_chunk<VEC>(p.x, p.xt, row * p.xs, c, p.d, h);
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] *= by;
    if (p.w1) {
        load_chunk<VEC>(p.w1, p.wt, 0, c, p.d, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] *= v[j];
    }
    if (p.gate_kind == GATE_CHANNEL || p.gate_kind == GATE_FULL) {
        load_chunk<VEC>(p.gate, p.gt, row * p.gs, c, p.d, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] *= v[j];
    }
    load_chunk<VEC>(p.res, p.rt, row * p.rs, c, p.d, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] = fmaf(v[j], p.res_scale, h[j]);
}

// A CTA a row, read three times (the second and third time from L2).
template <int VEC> __global__ void __launch_bounds__(1024) norm_pair_long_kernel(const PairParams p) {
    __shared__ float s_part[2][32];
    const uint32_t chunks = ((p.d + 127) / 128) * 16, n = blockDim.x;
    after_stream();
    let_next();
    uint32_t turn = 0; // of the two buffers of partial sums: a thread that is ahead by a sum writes the other
    for (uint64_t row = blockIdx.x; row < p.tokens; row += gridDim.x) {
        float by = p.scale;
        if (p.w1) {
            float sum = 0.0f;
            for (uint32_t c = threadIdx.x; c < chunks; c += n) {
                float v[8], part = 0.0f;
                load_chunk<VEC>(p.x, p.xt, row * p.xs, c, p.d, v);
#pragma unroll
                for (int j = 0; j < 8; ++j) part = fmaf(v[j], v[j], part);
                sum += part;
            }
            sum = team_sum<true>(sum, s_part[turn]);
            turn ^= 1u;
            by *= rsqrtf(sum / static_cast<float>(p.d) + p.eps);
        }
        if (p.gate_kind == GATE_TOKEN) by *= load1(p.gate, p.gt, row * p.gs);
        float root = 0.0f;
        if (p.y) {
            float sum = 0.0f;
            for (uint32_t c = threadIdx.x; c < chunks; c += n) {
                float h[8], part = 0.0f;
                pair_h<VEC>(p, row, c, by, h);
#pragma unroll
                for (int j = 0; j < 8; ++j) part = fmaf(h[j], h[j], part);
                sum += part;
            }
            sum = team_sum<true>(sum, s_part[turn]);
            turn ^= 1u;
            root = rsqrtf(sum / static_cast<float>(p.d) + p.eps);
        }
        // whole warps go round together: a scale's 16 lanes exchange inside
        for (uint32_t c0 = threadIdx.x & ~31u; c0 < chunks; c0 += n) {
            const uint32_t c = c0 + (threadIdx.x & 31u);
            float h[8], w[8];
            pair_h<VEC>(p, row, c, by, h);
            if (p.y) load_chunk<VEC>(p.w2, p.wt, 0, c, p.d, w);
            if (p.res_out) store_chunk<VEC>(p.res_out, p.rt, row * p.rs, c, p.d, h);
            if (!p.y) continue;
#pragma unroll
            for (int j = 0; j < 8; ++j) h[j] = h[j] * root * w[j];
            if (p.yt == FM_X_E4M3)
                store_e4m3<VEC>(p, row, c, h);
            else
                store_chunk<VEC>(p.y, p.yt, row * p.ys, c, p.d, h);
        }
    }
}

template <int VEC> int dispatch_pair(const PairParams &p, cudaStream_t s) {
    const uint32_t chunks = (p.d + 127) / 128 * 16, threads = chunks >= 1024 ? 1024 : (chunks + 31) / 32 * 32;
    const uint32_t most = static_cast<uint32_t>(device_sm_count()) * 8;
    return launch("norm_pair_long_kernel", norm_pair_long_kernel<VEC>,
                  {dim3(p.tokens < most ? p.tokens : most), threads, 0, 1}, s, p);
}

} // namespace
} // namespace fmb

using namespace fmb;

extern "C" int fmcuda_norm_add_norm(const fmcuda_norm_add_norm_args *a, void *stream) {
    if (!a) return set_error(FM_STATUS_INVALID_ARGUMENT, "null norm arguments");
    if (a->d_model == 0 || a->d_model > (1u << 24))
        return set_error(FM_STATUS_SHAPE_MISMATCH, "norm width must be 1 to 2^24");
    if (!is_float_x(a->x_dtype) || !is_float_x(a->residual_dtype) ||
        ((a->post_weight || a->pre_weight) && !is_float_x(a->weight_dtype)) || (a->gate && !is_float_x(a->gate_dtype)))
        return set_error(FM_STATUS_INVALID_ARGUMENT, "norm inputs must be float32, bfloat16 or float16");
    if (a->pre_weight && !is_float_x(a->y_dtype) && a->y_dtype != FM_X_E4M3)
        return set_error(FM_STATUS_INVALID_ARGUMENT, "norm output must be float32, bfloat16, float16 or e4m3");
    if (!(a->epsilon >= 0.0f)) return set_error(FM_STATUS_INVALID_ARGUMENT, "norm epsilon must not be negative");
    if (!std::isfinite(a->scale) || !std::isfinite(a->residual_scale))
        return set_error(FM_STATUS_INVALID_ARGUMENT, "norm scales must be finite");
    if (a->tokens == 0) return FM_STATUS_OK;
    if (!a->x || !a->residual || (a->pre_weight && !a->y) || (!a->pre_weight && !a->residual_out))
        return set_error(FM_STATUS_INVALID_ARGUMENT, "null norm buffer");
    const bool codes = a->pre_weight && a->y_dtype == FM_X_E4M3;
    if (codes && !a->scales) return set_error(FM_STATUS_INVALID_ARGUMENT, "an e4m3 output needs scales");
    if (!aligned_to_value(a->x, a->x_dtype) || !aligned_to_value(a->residual, a->residual_dtype) ||
        !aligned_to_value(a->residual_out, a->residual_dtype) ||
        ((a->post_weight || a->pre_weight) && (!aligned_to_value(a->post_weight, a->weight_dtype) ||
                                               !aligned_to_value(a->pre_weight, a->weight_dtype))) ||
        (a->gate && !aligned_to_value(a->gate, a->gate_dtype)) ||
        (a->pre_weight && !aligned_to_value(a->y, a->y_dtype)) || (codes && !aligned_to_value(a->scales, FM_X_F32)))
        return set_error(FM_STATUS_INVALID_ARGUMENT, "norm buffer is not aligned to its values");
    const int64_t d = a->d_model;
    const bool channels = a->gate && !a->gate_per_token;
    if (a->tokens > 1 && (a->x_stride < d || a->residual_stride < d || (a->pre_weight && a->y_stride < d)))
        return set_error(FM_STATUS_SHAPE_MISMATCH, "norm row stride is smaller than the row");
    if (a->gate && a->tokens > 1 && (a->gate_stride < 0 || (channels && a->gate_stride && a->gate_stride < d)))
        return set_error(FM_STATUS_SHAPE_MISMATCH, "gate row stride is negative or smaller than the row");
    const bool one_row = a->tokens == 1 || a->gate_stride == 0;
    PairParams p{};
    p.x = a->x;
    p.w1 = a->post_weight;
    p.gate = a->gate;
    p.res = a->residual;
    p.w2 = a->pre_weight;
    p.y = a->pre_weight ? a->y : nullptr;
    p.res_out = a->residual_out;
    p.scales = a->scales;
    p.xs = a->x_stride;
    p.gs = one_row ? 0 : a->gate_stride;
    p.rs = a->residual_stride;
    p.ys = a->y_stride;
    p.xt = a->x_dtype;
    p.rt = a->residual_dtype;
    p.wt = a->weight_dtype;
    p.gt = a->gate_dtype;
    p.yt = a->y_dtype;
    p.gate_kind = !a->gate ? GATE_NONE : !channels ? GATE_TOKEN : one_row ? GATE_CHANNEL : GATE_FULL;
    p.tokens = a->tokens;
    p.d = a->d_model;
    p.scale = a->scale;
    p.res_scale = a->residual_scale;
    p.eps = a->epsilon;
    auto fits = [&](int64_t values, uint32_t bytes) {
        auto at = [&](const void *q) { return reinterpret_cast<uintptr_t>(q) % bytes == 0; };
        auto row = [&](int64_t stride) { return a->tokens == 1 || stride % values == 0; };
        return d % values == 0 && row(p.xs) && row(p.rs) && (!p.y || (row(p.ys) && at(p.y))) && at(p.x) && at(p.res) &&
               at(p.res_out) && at(p.w1) && at(p.w2) && (!channels || (p.gs % values == 0 && at(p.gate)));
    };
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return fits(8, 16) ? dispatch_pair<8>(p, s) : fits(2, 8) ? dispatch_pair<2>(p, s) : dispatch_pair<1>(p, s);
}
