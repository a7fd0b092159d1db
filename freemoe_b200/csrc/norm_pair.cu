// norm_pair.cu -- the norms around a block: the norm of the block's output, its gated
// and scaled addition to the residual stream, and the norm before the next block.
//
//   n = x w1 / sqrt(mean(x^2) + eps),  h = a r + s g n,  y = h w2 / sqrt(mean(h^2) + eps)
//
// The operator is one read of x and r (and of a gate of their shape) and one write of h
// and y.  The second mean is of h itself, not of the four sums that would give it in one
// pass over x and r: where the block's output cancels the stream those lose all their
// digits.
//
// Measured, 8192 rows of 4096: bf16 46 us (268 MB, 5.8 TB/s, 89% of the rate of a copy), to
// e4m3 46, x in f32 58 (336 MB), x and y in f32 77 (403 MB), a gate of x's shape 54; rows of 8192
// 88; rows of 4095 82 (accesses of two bytes).  A row alone 3.1 us: a launch, the loads and two
// sums, one after the other.
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
    float scale, res_scale, eps, per_value; // per_value: 1 / d
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

// Rows longer than the registers of a CTA hold (16384 values): read three times, the second and third
// from L2.  1024 rows of 32768 in bf16 101 us (134 MB; 2048 rows of 16384, in registers, 54); one of
// 131072 44.
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
            by *= rsqrtf(sum * p.per_value + p.eps);
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
            root = rsqrtf(sum * p.per_value + p.eps);
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

// A chunk as it was loaded: nothing waits for the loads before get().  VEC 8: accesses of 16
// bytes, of a type that is known; otherwise (T is PAIR_ANY) of a type at run time, accesses of two
// values or one in the first words of their places.
constexpr int PAIR_ANY = -1;
template <int VEC, int T> struct PairChunk {
    uint32_t w[VEC != 8 || T == FM_X_F32 ? 8 : 4];
    __device__ __forceinline__ void load(const void *p, int32_t type, int64_t row, uint32_t c, uint32_t d) {
        const int32_t t = T == PAIR_ANY ? type : T;
        if constexpr (VEC == 8) {
            Raw8 q{};
            if (c * 8 < d) q = raw8_load(p, T, row + c * 8);
            const uint32_t all[8] = {q.a.x, q.a.y, q.a.z, q.a.w, q.b.x, q.b.y, q.b.z, q.b.w};
#pragma unroll
            for (uint32_t i = 0; i < sizeof(w) / 4; ++i) w[i] = all[i];
        } else {
            // the type is asked for once, not at each value (1700 rows of 311 9.3 -> 7.0 us, 8192 of 4095 92 -> 82)
            const char *base = static_cast<const char *>(p) + row * x_size(t);
            if (t == FM_X_F32) {
#pragma unroll
                for (int j = 0; j < 8; j += VEC) {
                    const uint32_t e = value_at<VEC>(c, j);
                    const uint32_t *at = reinterpret_cast<const uint32_t *>(base) + e;
                    uint2 v = make_uint2(0, 0);
                    if (e < d) {
                        if constexpr (VEC == 2)
                            v = *reinterpret_cast<const uint2 *>(at);
                        else
                            v.x = *at;
                    }
                    w[j] = v.x;
                    if constexpr (VEC == 2) w[j + 1] = v.y;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; j += VEC) {
                    const uint32_t e = value_at<VEC>(c, j);
                    const uint16_t *at = reinterpret_cast<const uint16_t *>(base) + e;
                    w[j] = 0;
                    if (e >= d) continue;
                    if constexpr (VEC == 2)
                        w[j] = *reinterpret_cast<const uint32_t *>(at);
                    else
                        w[j] = *at;
                }
            }
        }
    }
    __device__ __forceinline__ void get(int32_t type, float (&v)[8]) const {
        const int32_t t = T == PAIR_ANY ? type : T;
        if constexpr (VEC == 8) {
            constexpr int B = sizeof(w) == 32 ? 4 : 0; // (raw8_unpack looks at the second four with f32 only)
            raw8_unpack(Raw8{make_uint4(w[0], w[1], w[2], w[3]), make_uint4(w[B], w[B + 1], w[B + 2], w[B + 3])},
                        T, v);
        } else {
            if (t == FM_X_F32) {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(w[j]);
            } else if (t == FM_X_BF16) {
                values<__nv_bfloat16>(v);
            } else {
                values<__half>(v);
            }
        }
    }
    template <typename H> __device__ __forceinline__ void values(float (&v)[8]) const {
#pragma unroll
        for (int j = 0; j < 8; j += VEC) {
            const H *h = reinterpret_cast<const H *>(&w[j]);
            v[j] = static_cast<float>(h[0]);
            if constexpr (VEC == 2) v[j + 1] = static_cast<float>(h[1]);
        }
    }
};

// The sum over a team, for warps that come in fours (the others' places hold zeros): every thread
// adds up the partial sums itself.  (By shuffles they are another chain of five.)
template <bool CTA> __device__ __forceinline__ float pair_sum(float v, float4 *s_part) {
    v = warp_sum(v);
    if constexpr (CTA) {
        if ((threadIdx.x & 31u) == 0) reinterpret_cast<float *>(s_part)[threadIdx.x >> 5] = v;
        __syncthreads();
        v = 0.0f;
        for (uint32_t i = 0; i * 128 < blockDim.x; ++i) {
            const float4 q = s_part[i];
            v += (q.x + q.y) + (q.z + q.w);
        }
    }
    return v;
}

// A chunk of a weight, of a type at run time in each form.
template <int VEC> struct PairWeight {
    PairChunk<VEC == 8 ? 2 : VEC, PAIR_ANY> narrow;
    Raw8 wide;
    __device__ __forceinline__ void load(const void *p, int32_t t, uint32_t c, uint32_t d) {
        if constexpr (VEC == 8) {
            wide = Raw8{};
            if (c * 8 < d) wide = raw8_load(p, t, c * 8);
        } else {
            narrow.load(p, t, 0, c, d);
        }
    }
    __device__ __forceinline__ void get(int32_t t, float (&v)[8]) const {
        if constexpr (VEC == 8)
            raw8_unpack(wide, t, v);
        else
            narrow.get(t, v);
    }
};

// A team (see norm_rows.cuh) a row, whose values stay in registers between the two norms;
// the next row is on its way meanwhile (FULL: and a gate of the row's own).  The weights
// wait in shared memory as f32, the first one with the scale and a gate by channels in it.
// ONE: a CTA has one row, and a thread's weights come straight to its registers.
template <int VEC, int XT, int RT, bool FULL, bool CTA, bool ONE, int ITER, int MOST>
__global__ void __launch_bounds__(MOST, MOST == 512 && VEC == 8 && RT != FM_X_F32 ? 2 : 1) norm_pair_kernel(const PairParams p) {
    const uint32_t nt = CTA ? blockDim.x : 32u, teams = CTA ? 1u : blockDim.x / 32;
    // chunk c's first four values of w1 in s_w[c], the others, then w2's, `all` further each: lanes side
    // by side (with a chunk's eight together LDS takes twice as long, and 8192 x 4096 48 us)
    extern __shared__ float4 s_w[];
    __shared__ float4 s_part[2][8];
    const uint32_t c0 = CTA ? threadIdx.x : threadIdx.x % 32, all = nt * ITER;
    const uint64_t step = static_cast<uint64_t>(gridDim.x) * teams;
    after_stream();
    let_next();
    uint64_t row = CTA ? blockIdx.x : blockIdx.x * teams + threadIdx.x / 32;
    PairChunk<VEC, XT> x[ITER];
    PairChunk<VEC, RT> r[ITER];
    auto load = [&](uint64_t at) {
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            x[i].load(p.x, p.xt, at * p.xs, c0 + i * nt, p.d);
            r[i].load(p.res, p.rt, at * p.rs, c0 + i * nt, p.d);
        }
    };
    if (row < p.tokens) load(row);
    // chunk c of the first weight, with what is in it
    auto first_weight = [&](uint32_t c, float (&w)[8]) {
        float g[8];
        if (p.w1)
            load_chunk<VEC>(p.w1, p.wt, 0, c, p.d, w);
        else
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = 1.0f;
        if (p.gate_kind == GATE_CHANNEL) load_chunk<VEC>(p.gate, p.gt, 0, c, p.d, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] *= p.gate_kind == GATE_CHANNEL ? g[j] * p.scale : p.scale;
    };
    float w1[ONE ? ITER : 1][8], w2[ONE ? ITER : 1][8];
    if constexpr (ONE) { // all loads, then their values (one row of 4096: 3.05 -> 2.9 us)
        PairWeight<VEC> a, g, b;
        if (p.w1) a.load(p.w1, p.wt, c0, p.d);
        if (p.gate_kind == GATE_CHANNEL) g.load(p.gate, p.gt, c0, p.d);
        if (p.y) b.load(p.w2, p.wt, c0, p.d);
#pragma unroll
        for (int j = 0; j < 8; ++j) w1[0][j] = 1.0f, w2[0][j] = p.scale;
        if (p.w1) a.get(p.wt, w1[0]);
        if (p.gate_kind == GATE_CHANNEL) {
            g.get(p.gt, w2[0]);
#pragma unroll
            for (int j = 0; j < 8; ++j) w2[0][j] *= p.scale;
        }
        mul8(w1[0], w2[0]);
        if (p.y) b.get(p.wt, w2[0]);
    }
    for (uint32_t c = threadIdx.x; !ONE && c < all; c += blockDim.x) {
        float w[8];
        first_weight(c, w);
        s_w[c] = make_float4(w[0], w[1], w[2], w[3]);
        s_w[all + c] = make_float4(w[4], w[5], w[6], w[7]);
        if (!p.y) continue;
        load_chunk<VEC>(p.w2, p.wt, 0, c, p.d, w);
        s_w[2 * all + c] = make_float4(w[0], w[1], w[2], w[3]);
        s_w[3 * all + c] = make_float4(w[4], w[5], w[6], w[7]);
    }
    if (threadIdx.x < 16) s_part[threadIdx.x / 8][threadIdx.x % 8] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    __syncthreads();
    uint32_t turn = 0; // of the two buffers of partial sums: a thread that is ahead by a sum writes the other
    for (; row < p.tokens; row += step) {
        float h[ITER][8];
#pragma unroll
        for (int i = 0; i < ITER; ++i) x[i].get(p.xt, h[i]);
        PairChunk<VEC, RT> g[FULL ? ITER : 1];
        if constexpr (FULL) {
#pragma unroll
            for (int i = 0; i < ITER; ++i) g[i].load(p.gate, p.gt, row * p.gs, c0 + i * nt, p.d);
        }
        float by = 1.0f, token_gate = 1.0f;
        if (p.gate_kind == GATE_TOKEN) token_gate = load1(p.gate, p.gt, row * p.gs);
        if (p.w1) {
            uint64_t sums = 0;
#pragma unroll
            for (int i = 0; i < ITER; ++i) sums = squares8(h[i], sums);
            const float sum = pair_sum<CTA>(both(sums), s_part[turn]);
            turn ^= 1u;
            by = rsqrtf(sum * p.per_value + p.eps);
        }
        by *= token_gate;
        uint64_t sums = 0;
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const uint32_t c = c0 + i * nt;
            float v[8];
            mul8(h[i], by);
            if constexpr (ONE) {
                mul8(h[i], w1[i]);
            } else {
                const float4 wa = s_w[c], wb = s_w[all + c];
                const float w[8] = {wa.x, wa.y, wa.z, wa.w, wb.x, wb.y, wb.z, wb.w};
                mul8(h[i], w);
            }
            if constexpr (FULL) {
                g[i].get(p.gt, v);
                mul8(h[i], v);
            } else if (p.gate_kind == GATE_FULL) {
                load_chunk<VEC>(p.gate, p.gt, row * p.gs, c, p.d, v);
                mul8(h[i], v);
            }
            r[i].get(p.rt, v);
            add8(h[i], v, p.res_scale);
            sums = squares8(h[i], sums);
        }
        if (p.res_out) {
#pragma unroll
            for (int i = 0; i < ITER; ++i)
                store_chunk<VEC>(p.res_out, RT == PAIR_ANY ? p.rt : RT, row * p.rs, c0 + i * nt, p.d, h[i]);
        }
        // (right after this row's values were taken the loads cost more than they hide: 8192 x 4096 51 us, 46 here)
        if (!ONE && row + step < p.tokens) load(row + step);
        if (!p.y) continue;
        const float sum = pair_sum<CTA>(both(sums), s_part[turn]);
        turn ^= 1u;
        const float root = rsqrtf(sum * p.per_value + p.eps);
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const uint32_t c = c0 + i * nt;
            mul8(h[i], root);
            if constexpr (ONE) {
                mul8(h[i], w2[i]);
            } else {
                const float4 wa = s_w[2 * all + c], wb = s_w[3 * all + c];
                const float w[8] = {wa.x, wa.y, wa.z, wa.w, wb.x, wb.y, wb.z, wb.w};
                mul8(h[i], w);
            }
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

template <int VEC, int XT, int RT, bool FULL, bool CTA, bool ONE, int ITER, int MOST>
int launch_pair(const PairParams &p, uint32_t threads, cudaStream_t s) {
    auto kfn = norm_pair_kernel<VEC, XT, RT, FULL, CTA, ONE, ITER, MOST>;
    const uint32_t teams = CTA ? 1 : threads / 32, want = p.tokens / teams + (p.tokens % teams ? 1 : 0);
    const uint32_t smem = ONE ? 0 : (CTA ? threads : 32) * ITER * 64, most = ONE ? 0 : (CTA ? MOST : 32) * ITER * 64;
    uint32_t grid = static_cast<uint32_t>(device_sm_count());
    if (ONE) grid = want;
    // more rows than SMs: as many CTAs as the GPU holds; otherwise one a row
    if (want > grid) grid *= ctas_per_sm(kfn, {dim3(), threads, smem, 1, most});
    return launch("norm_pair_kernel", kfn, {dim3(want < grid ? want : grid), threads, smem, 1, most}, s, p);
}

// Short rows to warps, four a CTA; longer ones to CTAs, a thread two chunks, or one and a row a CTA
// where there are rows for half the threads of the GPU only (latency counts then: one row of 4096
// 3.4 -> 3.1 us, 256 rows 4.5 -> 4.1; but 512 rows of 4096 6.6 -> 7.1, 1024 9.1 -> 12.1).
template <int VEC, int XT, int RT, bool FULL = false> int dispatch_width(const PairParams &p, cudaStream_t s) {
    const uint32_t chunks = (p.d + 127) / 128 * 16, one = (chunks + 31) / 32 * 32, two = ((chunks + 1) / 2 + 31) / 32 * 32;
    const bool few = static_cast<uint64_t>(p.tokens) * one <= static_cast<uint64_t>(device_sm_count()) * 1024;
    if (p.d <= 256) return launch_pair<VEC, XT, RT, FULL, false, false, 1, 128>(p, 128, s);
    if (p.d <= 1024) return launch_pair<VEC, XT, RT, FULL, false, false, 4, 128>(p, 128, s);
    if (few && one <= 1024) {
        if constexpr (VEC != 8) {
            // code that runs once comes from memory: that of one pair of types is shorter (a row of 4095
            // in bf16 3.0 us; with many rows they take the same time).  The pairs here are a stream and its
            // block in one type, and a block in f32; the other four have types at run time, 4.4 to 4.9 us.
            auto typed = [&](int32_t xt, int32_t rt) { return p.xt == xt && p.rt == rt; };
            if (typed(FM_X_BF16, FM_X_BF16))
                return launch_pair<VEC, FM_X_BF16, FM_X_BF16, FULL, true, true, 1, 1024>(p, one, s);
            if (typed(FM_X_F32, FM_X_BF16))
                return launch_pair<VEC, FM_X_F32, FM_X_BF16, FULL, true, true, 1, 1024>(p, one, s);
            if (typed(FM_X_F16, FM_X_F16))
                return launch_pair<VEC, FM_X_F16, FM_X_F16, FULL, true, true, 1, 1024>(p, one, s);
            if (typed(FM_X_F32, FM_X_F16))
                return launch_pair<VEC, FM_X_F32, FM_X_F16, FULL, true, true, 1, 1024>(p, one, s);
            if (typed(FM_X_F32, FM_X_F32))
                return launch_pair<VEC, FM_X_F32, FM_X_F32, FULL, true, true, 1, 1024>(p, one, s);
        }
        return launch_pair<VEC, XT, RT, FULL, true, true, 1, 1024>(p, one, s);
    }
    if (two <= 512) return launch_pair<VEC, XT, RT, FULL, true, false, 2, 512>(p, two, s);
    if (two <= 1024) return launch_pair<VEC, XT, RT, FULL, true, false, 2, 1024>(p, two, s);
    const uint32_t most = static_cast<uint32_t>(device_sm_count()) * 2;
    return launch("norm_pair_long_kernel", norm_pair_long_kernel<VEC>,
                  {dim3(p.tokens < most ? p.tokens : most), 1024, 0, 1, 0}, s, p);
}

// A gate of x's shape has loads of its own where it is of the residual's type, 16 bits (8192 x 4096
// in bf16: 57 us, 65 where they come when they are needed).
template <int XT> int dispatch_residual(const PairParams &p, cudaStream_t s) {
    if (p.gate_kind == GATE_FULL && p.gt == p.rt) {
        if constexpr (XT != FM_X_F16)
            if (p.rt == FM_X_BF16) return dispatch_width<8, XT, FM_X_BF16, true>(p, s);
        if constexpr (XT != FM_X_BF16)
            if (p.rt == FM_X_F16) return dispatch_width<8, XT, FM_X_F16, true>(p, s);
    }
    if (p.rt == FM_X_BF16) return dispatch_width<8, XT, FM_X_BF16>(p, s);
    if (p.rt == FM_X_F16) return dispatch_width<8, XT, FM_X_F16>(p, s);
    return dispatch_width<8, XT, FM_X_F32>(p, s);
}

template <int VEC> int dispatch_pair(const PairParams &p, cudaStream_t s) {
    if constexpr (VEC != 8) {
        return dispatch_width<VEC, PAIR_ANY, PAIR_ANY>(p, s);
    } else {
        if (p.xt == FM_X_BF16) return dispatch_residual<FM_X_BF16>(p, s);
        if (p.xt == FM_X_F16) return dispatch_residual<FM_X_F16>(p, s);
        return dispatch_residual<FM_X_F32>(p, s);
    }
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
    p.per_value = 1.0f / static_cast<float>(a->d_model);
    auto fits = [&](int64_t values, uint32_t bytes) {
        auto at = [&](const void *q) { return reinterpret_cast<uintptr_t>(q) % bytes == 0; };
        auto row = [&](int64_t stride) { return a->tokens == 1 || stride % values == 0; };
        return d % values == 0 && row(p.xs) && row(p.rs) && (!p.y || (row(p.ys) && at(p.y))) && at(p.x) && at(p.res) &&
               at(p.res_out) && at(p.w1) && at(p.w2) && (!channels || (p.gs % values == 0 && at(p.gate)));
    };
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return fits(8, 16) ? dispatch_pair<8>(p, s) : fits(2, 8) ? dispatch_pair<2>(p, s) : dispatch_pair<1>(p, s);
}
