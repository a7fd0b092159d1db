// norm.cu -- root-mean-square norm of rows with the residual's addition, to
// f32 / bf16 / f16 or to e4m3 codes with one scale for each 128 values.
//
//   h = x + residual,  y = h * w / sqrt(mean(h^2) + eps)
//
// (the RMSNorm of Engine::forward_token, src/engine.cpp, whose sum is a double
// over one token; here f32 partial sums of at most 32 values a thread joined
// pairwise).  The operator is one read of x and residual and one write of y and
// h; the weight stays on the SM over the rows of a CTA.
//
// Measured, 8192 rows of 4096, bf16 with the residual, to 8 bits (236 MB): 40 to 44 us by
// machine, 84 to 91% of the rate of a copy; to bf16 (268 MB) 49 us, 85%; f32 throughout
// (537 MB) 96 us, 87%.  What it took: the next row's
// loads under way while a row is summed (61 -> 42), types fixed at compile time and
// quotients without a division (49 -> 40 with the issue slots 70% busy before).  Widths
// that are not whole eights: 4094 50 us, 4095 80 (bound by accesses of two bytes).
// One row: 2.4 us, latency.
#include <string>
#include <type_traits>

#include "launch.cuh"
#include "vec8.cuh"

namespace fmb {

namespace {

struct NormParams {
    const void *x, *res, *w;
    void *y, *res_out;
    float *scales;
    int64_t xs, rs, ys;
    int32_t xt, rt, wt, yt;
    uint32_t tokens, d;
    float eps;
};

// The sum over a team: a warp, or (CTA) all warps of the CTA.
template <bool CTA> __device__ __forceinline__ float team_sum(float v, float *s_part) {
    v = warp_sum(v);
    if constexpr (CTA) {
        const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
        if (lane == 0) s_part[warp] = v;
        __syncthreads();
        v = lane < blockDim.x / 32 ? s_part[lane] : 0.0f;
        v = warp_sum(v);
    }
    return v;
}

// A team (a warp, or the CTA) of n threads takes a row; its thread c
// holds chunks c, c + n, ... of 8 values.  VEC 8: a chunk is 8 consecutive
// values (16-byte accesses).  Otherwise the chunks of a group of 128 values are
// dealt out by VEC values (2, or 1) over 16 lanes, so that the accesses of the
// lanes still lie side by side.  Always 16 neighbouring lanes hold a scale's group.
template <int VEC> __device__ __forceinline__ uint32_t value_at(uint32_t c, int j) {
    return VEC == 8 ? c * 8 + j : (c >> 4) * 128 + j / VEC * (16 * VEC) + (c & 15u) * VEC + j % VEC;
}

template <int VEC>
__device__ __forceinline__ void load_chunk(const void *p, int32_t t, int64_t row, uint32_t c, uint32_t d,
                                           float (&v)[8]) {
    if constexpr (VEC == 8) {
        if (c * 8 < d) {
            raw8_unpack(raw8_load(p, t, row + c * 8), t, v);
            return;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.0f;
    } else if constexpr (VEC == 2) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const uint32_t e = value_at<VEC>(c, j);
            float2 f = make_float2(0.0f, 0.0f);
            if (e < d) f = load2(p, t, row + e);
            v[j] = f.x;
            v[j + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t e = value_at<VEC>(c, j);
            v[j] = e < d ? load1(p, t, row + e) : 0.0f;
        }
    }
}

template <int VEC>
__device__ __forceinline__ void store_chunk(void *p, int32_t t, int64_t row, uint32_t c, uint32_t d,
                                            const float (&v)[8]) {
    if constexpr (VEC == 8) {
        if (c * 8 < d) store8(p, t, row + c * 8, v);
    } else if constexpr (VEC == 2) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const uint32_t e = value_at<VEC>(c, j);
            if (e < d) store2(p, t, row + e, v[j], v[j + 1]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t e = value_at<VEC>(c, j);
            if (e < d) store1(p, t, row + e, v[j]);
        }
    }
}

// The 16 lanes of a group call this together; lanes past the row's end hold zeros.
template <int VEC>
__device__ __forceinline__ void store_e4m3(const NormParams &p, uint64_t row, uint32_t c, const float (&v)[8]) {
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(v[j]));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    // Quotients as a product with the reciprocal and one correction by the product's error,
    // which a fused operation gives exactly (Markstein, IBM J. Res. Dev. 34, 1990): correctly
    // rounded but for rare cases.  (A code is a rounding of its quotient: an error in the last
    // bit flips codes.)
    auto quotient = [](float x, float y, float inv) {
        const float q = x * inv;
        return fmaf(fmaf(-q, y, x), inv, q);
    };
    // An infinite scale has no correction (it would be infinity times zero): inv is 0 then, a
    // finite value by it 0 and an infinite one NaN, and with 0 for the divisor they stay so.
    const bool finite = top < INFINITY;
    const float scale = finite ? quotient(fmaxf(top, 1e-10f), 448.0f, 1.0f / 448.0f) : INFINITY;
    const float divisor = finite ? scale : 0.0f;
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(inv) : "f"(scale));
    auto code = [&](float x) { return quotient(x, divisor, inv); };
    uint8_t *y = static_cast<uint8_t *>(p.y) + row * p.ys;
    const uint32_t groups = (p.d + 127) / 128;
    if ((c & 15u) == 0 && (c >> 4) < groups) p.scales[row * groups + (c >> 4)] = scale;
    if constexpr (VEC == 8) {
        if (c * 8 < p.d) {
            uint32_t w[2];
#pragma unroll
            for (int i = 0; i < 2; ++i)
                w[i] = e4m3x2(code(v[4 * i]), code(v[4 * i + 1])) | e4m3x2(code(v[4 * i + 2]), code(v[4 * i + 3])) << 16;
            *reinterpret_cast<uint2 *>(y + c * 8) = make_uint2(w[0], w[1]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const uint32_t e = value_at<VEC>(c, j), two = e4m3x2(code(v[j]), code(v[j + 1]));
            if constexpr (VEC == 2) {
                if (e < p.d) *reinterpret_cast<uint16_t *>(y + e) = static_cast<uint16_t>(two);
            } else {
                const uint32_t next = value_at<VEC>(c, j + 1);
                if (e < p.d) y[e] = static_cast<uint8_t>(two);
                if (next < p.d) y[next] = static_cast<uint8_t>(two >> 8);
            }
        }
    }
}

// ITER chunks a thread, held in registers from the read to the write; the next row's
// are on their way while this one is summed and written.  The weight waits in shared
// memory, as f32 in the chunks' order.
// IN: the type of x and the residual, or NORM_ANY: at run time (VEC 8: with room for f32
// eights, which take two accesses; f32 has no variant of its own there).
constexpr int NORM_ANY = -1;

// A chunk as it was loaded, by accesses of VEC (1 or 2) values of type IN; nothing waits
// for the loads before get().
template <int VEC, int IN> struct RawChunk {
    static constexpr int N = 8 / VEC, BYTES = VEC * x_size(IN);
    using Word = std::conditional_t<BYTES == 8, uint2, std::conditional_t<BYTES == 4, uint32_t, uint16_t>>;
    Word w[N];
    __device__ __forceinline__ void load(const void *p, int64_t row, uint32_t c, uint32_t d) {
        const char *base = static_cast<const char *>(p) + row * x_size(IN);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint32_t e = value_at<VEC>(c, j * VEC);
            w[j] = Word{};
            if (e < d) w[j] = *reinterpret_cast<const Word *>(base + static_cast<uint64_t>(e) * x_size(IN));
        }
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if constexpr (VEC == 2) {
                const float2 f = load2(&w[j], IN, 0);
                v[2 * j] = f.x;
                v[2 * j + 1] = f.y;
            } else {
                v[j] = load1(&w[j], IN, 0);
            }
        }
    }
};

template <int VEC, int IN, int ITER> struct NormRow {
    static constexpr bool WIDE = VEC == 8 && IN == NORM_ANY, RAW = VEC != 8 && IN != NORM_ANY;
    uint4 x[ITER], r[ITER]; // VEC 8
    uint4 x2[WIDE ? ITER : 1], r2[WIDE ? ITER : 1];
    RawChunk<RAW ? VEC : 1, RAW ? IN : FM_X_F32> wx[RAW ? ITER : 1], wr[RAW ? ITER : 1];
    float h[ITER][8]; // types at run time, and not eights: already h

    __device__ __forceinline__ void load(const NormParams &p, uint64_t row, uint32_t c0, uint32_t step) {
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const uint32_t c = c0 + i * step;
            if constexpr (VEC == 8) {
                x[i] = r[i] = make_uint4(0, 0, 0, 0);
                if (WIDE) x2[i] = r2[i] = make_uint4(0, 0, 0, 0);
                if (c * 8 < p.d) {
                    if constexpr (WIDE) {
                        const Raw8 a = raw8_load(p.x, p.xt, row * p.xs + c * 8);
                        x[i] = a.a;
                        x2[i] = a.b;
                        if (p.res) {
                            const Raw8 b = raw8_load(p.res, p.rt, row * p.rs + c * 8);
                            r[i] = b.a;
                            r2[i] = b.b;
                        }
                    } else {
                        x[i] = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p.x) + row * p.xs + c * 8);
                        if (p.res)
                            r[i] = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p.res) + row * p.rs +
                                                                    c * 8);
                    }
                }
            } else if constexpr (RAW) {
                wx[i].load(p.x, row * p.xs, c, p.d);
                if (p.res) wr[i].load(p.res, row * p.rs, c, p.d);
            } else {
                load_chunk<VEC>(p.x, p.xt, row * p.xs, c, p.d, h[i]);
                if (p.res) {
                    float v[8];
                    load_chunk<VEC>(p.res, p.rt, row * p.rs, c, p.d, v);
#pragma unroll
                    for (int j = 0; j < 8; ++j) h[i][j] += v[j];
                }
            }
        }
    }
    __device__ __forceinline__ void get(const NormParams &p, float (&out)[ITER][8]) const {
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            if constexpr (VEC == 8) {
                raw8_unpack(Raw8{x[i], x2[WIDE ? i : 0]}, WIDE ? p.xt : IN, out[i]);
                if (p.res) {
                    float v[8];
                    raw8_unpack(Raw8{r[i], r2[WIDE ? i : 0]}, WIDE ? p.rt : IN, v);
#pragma unroll
                    for (int j = 0; j < 8; ++j) out[i][j] += v[j];
                }
            } else if constexpr (RAW) {
                wx[i].get(out[i]);
                if (p.res) {
                    float v[8];
                    wr[i].get(v);
#pragma unroll
                    for (int j = 0; j < 8; ++j) out[i][j] += v[j];
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) out[i][j] = h[i][j];
            }
        }
    }
};

template <int VEC, int IN, bool CTA, int ITER, int MOST>
__global__ void __launch_bounds__(MOST) add_rms_norm_kernel(const NormParams p) {
    const uint32_t nt = CTA ? blockDim.x : 32u, teams = CTA ? 1u : blockDim.x / 32;
    extern __shared__ float4 s_w[]; // chunk c: s_w[2 c], s_w[2 c + 1]
    __shared__ float s_part[2][32];
    const uint32_t c0 = CTA ? threadIdx.x : threadIdx.x % 32;
    const uint32_t team = CTA ? blockIdx.x : blockIdx.x * teams + threadIdx.x / 32;
    const uint64_t step = static_cast<uint64_t>(gridDim.x) * teams;
    after_stream();
    let_next();
    uint64_t row = team;
    NormRow<VEC, IN, ITER> next;
    if (row < p.tokens) next.load(p, row, c0, nt);
    for (uint32_t c = threadIdx.x; c < nt * ITER; c += blockDim.x) {
        float w[8];
        load_chunk<VEC>(p.w, p.wt, 0, c, p.d, w);
        s_w[2 * c] = make_float4(w[0], w[1], w[2], w[3]);
        s_w[2 * c + 1] = make_float4(w[4], w[5], w[6], w[7]);
    }
    __syncthreads();
    for (uint32_t turn = 0; row < p.tokens; row += step, turn ^= 1u) {
        float h[ITER][8];
        next.get(p, h);
        if (row + step < p.tokens) next.load(p, row + step, c0, nt);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < ITER; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) sum = fmaf(h[i][j], h[i][j], sum);
        // two buffers of partial sums: a thread that is ahead by a row writes the other one
        sum = team_sum<CTA>(sum, s_part[turn]);
        const float root = rsqrtf(sum / static_cast<float>(p.d) + p.eps);
        if (p.res_out) {
#pragma unroll
            for (int i = 0; i < ITER; ++i) 
                store_chunk<VEC>(p.res_out, IN == NORM_ANY ? p.rt : IN, row * p.rs, c0 + i * nt, p.d, h[i]);
        }
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const uint32_t c = c0 + i * nt;
            const float4 wa = s_w[2 * c], wb = s_w[2 * c + 1];
            const float w[8] = {wa.x, wa.y, wa.z, wa.w, wb.x, wb.y, wb.z, wb.w};
#pragma unroll
            for (int j = 0; j < 8; ++j) h[i][j] = h[i][j] * root * w[j];
            // one branch on the type, not one for each value
            if (p.yt == FM_X_E4M3)
                store_e4m3<VEC>(p, row, c, h[i]);
            else if (p.yt == FM_X_F32)
                store_chunk<VEC>(p.y, FM_X_F32, row * p.ys, c, p.d, h[i]);
            else if (p.yt == FM_X_BF16)
                store_chunk<VEC>(p.y, FM_X_BF16, row * p.ys, c, p.d, h[i]);
            else
                store_chunk<VEC>(p.y, FM_X_F16, row * p.ys, c, p.d, h[i]);
        }
    }
}

// Rows longer than the registers of a CTA hold: read twice, the second time from L2.
template <int VEC> __global__ void __launch_bounds__(1024) add_rms_norm_long_kernel(const NormParams p) {
    __shared__ float s_part[2][32];
    const uint32_t chunks = ((p.d + 127) / 128) * 16;
    after_stream();
    let_next();
    uint32_t turn = 0;
    for (uint64_t row = blockIdx.x; row < p.tokens; row += gridDim.x, turn ^= 1u) {
        float sum = 0.0f;
        for (uint32_t c = threadIdx.x; c < chunks; c += 1024) {
            float h[8], r[8];
            load_chunk<VEC>(p.x, p.xt, row * p.xs, c, p.d, h);
            if (p.res) {
                load_chunk<VEC>(p.res, p.rt, row * p.rs, c, p.d, r);
#pragma unroll
                for (int j = 0; j < 8; ++j) h[j] += r[j];
            }
            float part = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) part = fmaf(h[j], h[j], part);
            sum += part;
        }
        sum = team_sum<true>(sum, s_part[turn]);
        const float root = rsqrtf(sum / static_cast<float>(p.d) + p.eps);
        // whole warps go round together: a scale's 16 lanes exchange inside
        for (uint32_t c0 = threadIdx.x & ~31u; c0 < chunks; c0 += 1024) {
            const uint32_t c = c0 + (threadIdx.x & 31u);
            float h[8], r[8], w[8];
            load_chunk<VEC>(p.x, p.xt, row * p.xs, c, p.d, h);
            load_chunk<VEC>(p.w, p.wt, 0, c, p.d, w);
            if (p.res) {
                load_chunk<VEC>(p.res, p.rt, row * p.rs, c, p.d, r);
#pragma unroll
                for (int j = 0; j < 8; ++j) h[j] += r[j];
            }
            if (p.res_out) store_chunk<VEC>(p.res_out, p.rt, row * p.rs, c, p.d, h);
#pragma unroll
            for (int j = 0; j < 8; ++j) h[j] = h[j] * root * w[j];
            if (p.yt == FM_X_E4M3)
                store_e4m3<VEC>(p, row, c, h);
            else
                store_chunk<VEC>(p.y, p.yt, row * p.ys, c, p.d, h);
        }
    }
}

template <int VEC, int IN, bool CTA, int ITER, int MOST>
int launch_norm(const NormParams &p, uint32_t threads, cudaStream_t s) {
    auto kfn = add_rms_norm_kernel<VEC, IN, CTA, ITER, MOST>;
    const uint32_t teams = CTA ? 1 : threads / 32, want = (p.tokens + teams - 1) / teams;
    const uint32_t smem = (CTA ? threads : 32) * ITER * 32;
    uint32_t grid = static_cast<uint32_t>(device_sm_count());
    if (want > grid) { // as many CTAs as the GPU holds; otherwise one a row
        int per_sm = 0;
        if (smem > 48 * 1024) cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kfn, threads, smem) != cudaSuccess || per_sm < 1) {
            (void)cudaGetLastError();
            per_sm = 1;
        }
        grid *= static_cast<uint32_t>(per_sm);
    }
    return launch("add_rms_norm_kernel", kfn, {dim3(want < grid ? want : grid), threads, smem, 1}, s, p);
}

// Short rows to warps, four a CTA; longer ones to CTAs, a thread two chunks, or one where
// there are rows for half the threads of the GPU only (latency counts then).
template <int VEC, int IN> int dispatch_width(const NormParams &p, cudaStream_t s) {
    const uint32_t chunks = (p.d + 127) / 128 * 16, one = (chunks + 31) / 32 * 32, two = ((chunks + 1) / 2 + 31) / 32 * 32;
    const bool few = static_cast<uint64_t>(p.tokens) * one <= static_cast<uint64_t>(device_sm_count()) * 1024;
    if (p.d <= 256) return launch_norm<VEC, IN, false, 1, 128>(p, 128, s);
    if (p.d <= 1024) return launch_norm<VEC, IN, false, 4, 128>(p, 128, s);
    if (few && one <= 1024) return launch_norm<VEC, IN, true, 1, 1024>(p, one, s);
    if (two <= 512) return launch_norm<VEC, IN, true, 2, 512>(p, two, s);
    if (two <= 1024) return launch_norm<VEC, IN, true, 2, 1024>(p, two, s);
    const uint32_t most = static_cast<uint32_t>(device_sm_count()) * 2;
    return launch("add_rms_norm_long_kernel", add_rms_norm_long_kernel<VEC>,
                  {dim3(p.tokens < most ? p.tokens : most), 1024, 0, 1}, s, p);
}

template <int VEC> int dispatch_norm(const NormParams &p, cudaStream_t s) {
    const bool one_type = !(p.res || p.res_out) || p.xt == p.rt;
    if (one_type && p.xt == FM_X_BF16) return dispatch_width<VEC, FM_X_BF16>(p, s);
    if (one_type && p.xt == FM_X_F16) return dispatch_width<VEC, FM_X_F16>(p, s);
    if constexpr (VEC != 8)
        if (one_type) return dispatch_width<VEC, FM_X_F32>(p, s);
    return dispatch_width<VEC, NORM_ANY>(p, s);
}

} // namespace
} // namespace fmb

using namespace fmb;

extern "C" int fmcuda_add_rms_norm(const fmcuda_rms_norm_args *a, void *stream) {
    if (!a) return set_error(FM_STATUS_INVALID_ARGUMENT, "null norm arguments");
    if (a->d_model == 0 || a->d_model > (1u << 24))
        return set_error(FM_STATUS_SHAPE_MISMATCH, "norm width must be 1 to 2^24");
    if (!is_float_x(a->x_dtype) || !is_float_x(a->weight_dtype) ||
        ((a->residual || a->residual_out) && !is_float_x(a->residual_dtype)))
        return set_error(FM_STATUS_INVALID_ARGUMENT, "norm inputs must be float32, bfloat16 or float16");
    if (!is_float_x(a->y_dtype) && a->y_dtype != FM_X_E4M3)
        return set_error(FM_STATUS_INVALID_ARGUMENT, "norm output must be float32, bfloat16, float16 or e4m3");
    if (!(a->epsilon >= 0.0f)) return set_error(FM_STATUS_INVALID_ARGUMENT, "norm epsilon must not be negative");
    if (a->tokens == 0) return FM_STATUS_OK;
    if (!a->x || !a->weight || !a->y) return set_error(FM_STATUS_INVALID_ARGUMENT, "null norm buffer");
    if (a->y_dtype == FM_X_E4M3 && !a->scales)
        return set_error(FM_STATUS_INVALID_ARGUMENT, "an e4m3 output needs scales");
    if (!aligned_to_value(a->x, a->x_dtype) || !aligned_to_value(a->residual, a->residual_dtype) ||
        !aligned_to_value(a->residual_out, a->residual_dtype) || !aligned_to_value(a->weight, a->weight_dtype) ||
        !aligned_to_value(a->y, a->y_dtype) || !aligned_to_value(a->scales, FM_X_F32))
        return set_error(FM_STATUS_INVALID_ARGUMENT, "norm buffer is not aligned to its values");
    const int64_t d = a->d_model;
    if (a->tokens > 1 && (a->x_stride < d || a->y_stride < d ||
                          ((a->residual || a->residual_out) && a->residual_stride < d)))
        return set_error(FM_STATUS_SHAPE_MISMATCH, "norm row stride is smaller than the row");
    const NormParams p{a->x,        a->residual,        a->weight,   a->y,       a->residual_out,  a->scales,
                       a->x_stride, a->residual_stride, a->y_stride, a->x_dtype, a->residual_dtype, a->weight_dtype,
                       a->y_dtype,  a->tokens,          a->d_model,  a->epsilon};
    auto fits = [&](int64_t values, uint32_t bytes) {
        auto at = [&](const void *q) { return reinterpret_cast<uintptr_t>(q) % bytes == 0; };
        return d % values == 0 && a->x_stride % values == 0 && a->y_stride % values == 0 &&
               a->residual_stride % values == 0 && at(a->x) && at(a->residual) && at(a->weight) && at(a->y) &&
               at(a->residual_out);
    };
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return fits(8, 16) ? dispatch_norm<8>(p, s) : fits(2, 8) ? dispatch_norm<2>(p, s) : dispatch_norm<1>(p, s);
}
