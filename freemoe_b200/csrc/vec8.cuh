// vec8.cuh -- eight consecutive activation values as 16-byte accesses, for the
// bandwidth-bound kernels whose element types are run-time arguments (the
// branch on the type is uniform over the grid).
#pragma once

#include "common.cuh"

namespace fmb {

__host__ __device__ constexpr uint32_t x_size(int32_t dtype) {
    return dtype == FM_X_F32 ? 4u : dtype == FM_X_E4M3 ? 1u : 2u;
}

// The raw bytes of eight values: both words of a f32 eight, the first of a 16-bit one.
struct Raw8 {
    uint4 a, b;
};

// Eight values from element `at` on; 16-byte aligned.  Not through the read-only
// path: outputs may lie on inputs.
__device__ __forceinline__ Raw8 raw8_load(const void *p, int32_t dtype, uint64_t at) {
    Raw8 r;
    r.b = make_uint4(0, 0, 0, 0);
    if (dtype == FM_X_F32) {
        const uint4 *q = reinterpret_cast<const uint4 *>(static_cast<const float *>(p) + at);
        r.a = q[0];
        r.b = q[1];
    } else {
        r.a = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p) + at);
    }
    return r;
}

__device__ __forceinline__ void raw8_unpack(const Raw8 &r, int32_t dtype, float (&v)[8]) {
    const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w}; // (b: f32 only)
    if (dtype == FM_X_F32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
    } else if (dtype == FM_X_BF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi, int32_t dtype) {
    if (dtype == FM_X_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}

__device__ __forceinline__ void store8(void *p, int32_t dtype, uint64_t at, const float (&v)[8]) {
    if (dtype == FM_X_F32) {
        float4 *q = reinterpret_cast<float4 *>(static_cast<float *>(p) + at);
        q[0] = make_float4(v[0], v[1], v[2], v[3]);
        q[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else if (dtype == FM_X_BF16) {
        *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p) + at) =
            make_uint4(pack2(v[0], v[1], FM_X_BF16), pack2(v[2], v[3], FM_X_BF16), pack2(v[4], v[5], FM_X_BF16),
                       pack2(v[6], v[7], FM_X_BF16));
    } else {
        *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p) + at) =
            make_uint4(pack2(v[0], v[1], FM_X_F16), pack2(v[2], v[3], FM_X_F16), pack2(v[4], v[5], FM_X_F16),
                       pack2(v[6], v[7], FM_X_F16));
    }
}

// One value, for rows that 16-byte accesses do not fit.
__device__ __forceinline__ float load1(const void *p, int32_t dtype, uint64_t at) {
    if (dtype == FM_X_F32) return static_cast<const float *>(p)[at];
    const uint16_t w = static_cast<const uint16_t *>(p)[at];
    return dtype == FM_X_BF16 ? bf16_bits_to_f32(w) : fp16_bits_to_f32(w);
}

__device__ __forceinline__ void store1(void *p, int32_t dtype, uint64_t at, float v) {
    if (dtype == FM_X_F32)
        static_cast<float *>(p)[at] = v;
    else if (dtype == FM_X_BF16)
        static_cast<__nv_bfloat16 *>(p)[at] = __float2bfloat16_rn(v);
    else
        static_cast<__half *>(p)[at] = __float2half_rn(v);
}

// Two values, where their pairs are aligned.
__device__ __forceinline__ float2 load2(const void *p, int32_t dtype, uint64_t at) {
    if (dtype == FM_X_F32) return *reinterpret_cast<const float2 *>(static_cast<const float *>(p) + at);
    const uint32_t w = *reinterpret_cast<const uint32_t *>(static_cast<const uint16_t *>(p) + at);
    if (dtype == FM_X_BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}

__device__ __forceinline__ void store2(void *p, int32_t dtype, uint64_t at, float lo, float hi) {
    if (dtype == FM_X_F32)
        *reinterpret_cast<float2 *>(static_cast<float *>(p) + at) = make_float2(lo, hi);
    else
        *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(p) + at) = pack2(lo, hi, dtype);
}

// Two e4m3 codes, `lo` in the low byte; round to nearest even, largest 448, NaN kept.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

inline bool is_x16(int32_t dtype) { return dtype == FM_X_BF16 || dtype == FM_X_F16; }
inline bool is_float_x(int32_t dtype) { return dtype == FM_X_F32 || is_x16(dtype); }
// A null pointer is aligned.
inline bool aligned_to_value(const void *p, int32_t dtype) {
    return reinterpret_cast<uintptr_t>(p) % x_size(dtype) == 0;
}
inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

} // namespace fmb
