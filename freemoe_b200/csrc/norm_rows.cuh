// norm_rows.cuh -- what the kernels that norm rows share: how a row's values are dealt
// out to a team of threads, their loads and stores, sums over the team, and the
// rounding to e4m3 codes with one scale for each 128 values.
#pragma once

#include "ptx.cuh"
#include "vec8.cuh"

namespace fmb {

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
// P: the kernel's parameters, with the codes y, their row stride ys, the scales and the width d.
template <int VEC, typename P>
__device__ __forceinline__ void store_e4m3(const P &p, uint64_t row, uint32_t c, const float (&v)[8]) {
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

} // namespace fmb
