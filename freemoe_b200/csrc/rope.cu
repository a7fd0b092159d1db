// rope.cu -- rotary positions of new queries and keys, and the write of new
// keys and values into the pages of a cache.
//
//   (a, b) -> (a cos t - b sin t, a sin t + b cos t),  t = position * inv_freq[i]
//
// (src/rope.cpp of the reference turns one head at a time on the host).  The
// operator is one read of q, k and v and one write of q and of two cache rows a
// token; the cosines of a token are shared by all of its heads.  A CTA takes a
// token, or a part of its heads when there are too few tokens to fill the GPU.
//
// The angle of a far position does not fit f32 (at position 2^17 its last bit
// is 2^-7 radians), so the product is taken in turns in 64 bits, its whole part
// dropped, and only the fraction of a turn goes to f32: three 64-bit operations
// a pair, once for all heads.
#include <cmath>
#include <string>

#include "vec8.cuh"

namespace fmb {
namespace {

constexpr uint32_t ROPE_THREADS = 256;
constexpr uint32_t ROPE_MAX_DIM = 1024;

struct RopeParams {
    const void *q, *k, *v;
    void *q_out, *kc, *vc;
    const int32_t *positions;
    const int64_t *slots;
    const float *inv_freq;
    int64_t qt, qh, kt, kh, vt, vh, ot, oh, cp, ch, cr;
    int32_t in_t, out_t;
    uint32_t heads, kv_heads, dim, rot;
    float factor;
    uint32_t page_size;
    uint64_t n_slots;
    uint32_t head_items, value_items, items; // work items of a rotated head, of a value head, of a token
    int *status;
};

struct Place {
    const void *src;
    void *dst;
    int64_t from, to;
    uint32_t item;
    bool turns, live;
};

// Where item `it` of token `t` reads and writes: the heads of q, of k, of v in turn.
__device__ __forceinline__ Place rope_place(const RopeParams &p, uint32_t it, int64_t t, int64_t cache_row) {
    Place w;
    const uint32_t turned = (p.heads + p.kv_heads) * p.head_items;
    w.turns = it < turned;
    w.live = true;
    if (w.turns) {
        uint32_t h = it / p.head_items;
        w.item = it - h * p.head_items;
        if (h < p.heads) {
            w.src = p.q;
            w.dst = p.q_out;
            w.from = t * p.qt + h * p.qh;
            w.to = t * p.ot + h * p.oh;
            return w;
        }
        h -= p.heads;
        w.src = p.k;
        w.dst = p.kc;
        w.from = t * p.kt + h * p.kh;
        w.to = cache_row + h * p.ch;
    } else {
        const uint32_t h = (it - turned) / p.value_items;
        w.item = it - turned - h * p.value_items;
        w.src = p.v;
        w.dst = p.vc;
        w.from = t * p.vt + h * p.vh;
        w.to = cache_row + h * p.ch;
    }
    w.live = cache_row >= 0;
    return w;
}

// VEC: an item is 8 values and, for pairs at (i, i + rot/2), their 8 partners
// (heads, strides and rot/2 in whole eights).  Otherwise it is one pair or one
// value; consecutive lanes then take consecutive pairs.
template <bool VEC, bool INTER>
__global__ void __launch_bounds__(ROPE_THREADS) rope_append_kernel(const RopeParams p) {
    __shared__ float2 s_turn[ROPE_MAX_DIM / 2];
    const int64_t t = blockIdx.x;
    const uint32_t half = p.rot / 2;
    for (uint32_t i = threadIdx.x; i < half; i += blockDim.x) {
        const double turns = static_cast<double>(p.positions[t]) * static_cast<double>(p.inv_freq[i]) *
                             0.15915494309189533577; // 1 / (2 pi)
        float sn, cs;
        sincospif(2.0f * static_cast<float>(turns - rint(turns)), &sn, &cs);
        s_turn[i] = make_float2(cs * p.factor, sn * p.factor);
    }
    int64_t cache_row = -1;
    if (p.kc) {
        const int64_t slot = p.slots[t];
        if (slot >= 0 && static_cast<uint64_t>(slot) < p.n_slots) {
            const int64_t page = slot / p.page_size;
            cache_row = page * p.cp + (slot - page * p.page_size) * p.cr;
        } else if (slot >= 0 && threadIdx.x == 0 && blockIdx.y == 0) {
            raise_device_status(p.status, FM_STATUS_INVALID_ARGUMENT);
        }
    }
    __syncthreads();
    for (uint32_t it = blockIdx.y * blockDim.x + threadIdx.x; it < p.items; it += gridDim.y * blockDim.x) {
        const Place w = rope_place(p, it, t, cache_row);
        if (!w.live) continue;
        if constexpr (VEC) {
            float a[8], b[8];
            if (!w.turns) {
                raw8_unpack(raw8_load(w.src, p.in_t, w.from + w.item * 8), p.in_t, a);
                store8(w.dst, p.out_t, w.to + w.item * 8, a);
            } else if (INTER) {
                const uint32_t i0 = w.item * 4;
                raw8_unpack(raw8_load(w.src, p.in_t, w.from + w.item * 8), p.in_t, a);
                if (i0 < half) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 cs = s_turn[i0 + j];
                        b[2 * j] = a[2 * j] * cs.x - a[2 * j + 1] * cs.y;
                        b[2 * j + 1] = a[2 * j] * cs.y + a[2 * j + 1] * cs.x;
                    }
                    store8(w.dst, p.out_t, w.to + w.item * 8, b);
                } else {
                    store8(w.dst, p.out_t, w.to + w.item * 8, a);
                }
            } else if (w.item * 8 < half) {
                const uint32_t i0 = w.item * 8;
                raw8_unpack(raw8_load(w.src, p.in_t, w.from + i0), p.in_t, a);
                raw8_unpack(raw8_load(w.src, p.in_t, w.from + half + i0), p.in_t, b);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float2 cs = s_turn[i0 + j];
                    const float x = a[j] * cs.x - b[j] * cs.y;
                    b[j] = a[j] * cs.y + b[j] * cs.x;
                    a[j] = x;
                }
                store8(w.dst, p.out_t, w.to + i0, a);
                store8(w.dst, p.out_t, w.to + half + i0, b);
            } else {
                const uint32_t e = w.item * 8 + half; // behind the pairs
                raw8_unpack(raw8_load(w.src, p.in_t, w.from + e), p.in_t, a);
                store8(w.dst, p.out_t, w.to + e, a);
            }
        } else {
            if (w.turns && w.item < half) {
                const uint32_t ea = INTER ? 2 * w.item : w.item, eb = INTER ? ea + 1 : ea + half;
                const float a = load1(w.src, p.in_t, w.from + ea), b = load1(w.src, p.in_t, w.from + eb);
                const float2 cs = s_turn[w.item];
                store1(w.dst, p.out_t, w.to + ea, a * cs.x - b * cs.y);
                store1(w.dst, p.out_t, w.to + eb, a * cs.y + b * cs.x);
            } else {
                const uint32_t e = w.turns ? w.item + half : w.item;
                store1(w.dst, p.out_t, w.to + e, load1(w.src, p.in_t, w.from + e));
            }
        }
    }
}

} // namespace
} // namespace fmb

using namespace fmb;

extern "C" int fmcuda_rope_frequencies(uint32_t rot_dim, double base, const fmcuda_rope_scaling *sc, float *inv_freq,
                                       float *attention_factor) {
    if (!inv_freq || !attention_factor) return set_error(FM_STATUS_INVALID_ARGUMENT, "null rotary output");
    if (rot_dim == 0 || rot_dim % 2 || rot_dim > ROPE_MAX_DIM)
        return set_error(FM_STATUS_SHAPE_MISMATCH, "rotary width must be even, 2 to 1024");
    const int kind = sc ? sc->kind : FM_ROPE_PLAIN;
    if (!(base > 1.0) || !std::isfinite(base)) return set_error(FM_STATUS_INVALID_ARGUMENT, "rotary base must exceed 1");
    if (kind < FM_ROPE_PLAIN || kind > FM_ROPE_BANDS)
        return set_error(FM_STATUS_INVALID_ARGUMENT, "unknown rotary scaling");
    if (kind != FM_ROPE_PLAIN && !(sc->factor > 0.0 && std::isfinite(sc->factor)))
        return set_error(FM_STATUS_INVALID_ARGUMENT, "rotary scaling factor must be positive");
    const bool banded = kind == FM_ROPE_RAMP || kind == FM_ROPE_BANDS;
    if (banded && !(sc->trained_context > 0.0 && sc->slow > 0.0 && sc->fast > sc->slow))
        return set_error(FM_STATUS_INVALID_ARGUMENT, "rotary scaling needs a trained context and fast > slow > 0");
    if (kind == FM_ROPE_BASE && rot_dim == 2)
        return set_error(FM_STATUS_SHAPE_MISMATCH, "a scaled base needs a rotary width above 2");
    const double pi2 = 6.283185307179586476925, n = rot_dim;
    if (kind == FM_ROPE_BASE) base *= std::pow(sc->factor, n / (n - 2.0));
    // the pair that turns `turns` times in the trained context
    auto pair_of = [&](double turns) {
        return n * std::log(sc->trained_context / (turns * pi2)) / (2.0 * std::log(base));
    };
    double first = 0.0, last = 0.0;
    if (kind == FM_ROPE_RAMP) {
        first = std::fmax(std::floor(pair_of(sc->fast)), 0.0);
        last = std::fmin(std::ceil(pair_of(sc->slow)), n - 1.0);
        if (last <= first) last = first + 0.001; // a step instead of a ramp
    }
    for (uint32_t i = 0; i < rot_dim / 2; ++i) {
        double f = std::pow(base, -2.0 * i / n);
        if (kind == FM_ROPE_LINEAR) {
            f /= sc->factor;
        } else if (banded) {
            const double keep = kind == FM_ROPE_RAMP
                                    ? 1.0 - (i - first) / (last - first)
                                    : (sc->trained_context * f / pi2 - sc->slow) / (sc->fast - sc->slow);
            const double part = std::fmin(std::fmax(keep, 0.0), 1.0);
            f = part * f + (1.0 - part) * f / sc->factor;
        }
        inv_freq[i] = static_cast<float>(f);
    }
    *attention_factor =
        kind == FM_ROPE_RAMP && sc->factor > 1.0 ? static_cast<float>(0.1 * std::log(sc->factor) + 1.0) : 1.0f;
    return FM_STATUS_OK;
}

extern "C" int fmcuda_rope_append(const fmcuda_rope_append_args *a, void *stream) {
    if (!a) return set_error(FM_STATUS_INVALID_ARGUMENT, "null rotary arguments");
    if (a->heads == 0 || a->head_dim == 0 || a->head_dim > ROPE_MAX_DIM || a->heads > 65535 || a->kv_heads > 65535)
        return set_error(FM_STATUS_SHAPE_MISMATCH, "heads must be 1 to 65535 and head_dim 1 to 1024");
    if (a->rot_dim % 2 || a->rot_dim > a->head_dim)
        return set_error(FM_STATUS_SHAPE_MISMATCH, "rot_dim must be even and at most head_dim");
    if (!is_float_x(a->in_dtype) || !is_float_x(a->out_dtype))
        return set_error(FM_STATUS_INVALID_ARGUMENT, "rotary types must be float32, bfloat16 or float16");
    const bool cached = a->k || a->v || a->k_cache || a->v_cache;
    if (cached && (!a->k || !a->v || !a->k_cache || !a->v_cache || !a->slots))
        return set_error(FM_STATUS_INVALID_ARGUMENT, "k, v, their caches and slots come together");
    if (cached && (a->kv_heads == 0 || a->page_size == 0))
        return set_error(FM_STATUS_SHAPE_MISMATCH, "a cache has at least one head and one row a page");
    if (a->tokens == 0) return FM_STATUS_OK;
    if (!a->q || !a->q_out || !a->positions || (a->rot_dim && !a->inv_freq))
        return set_error(FM_STATUS_INVALID_ARGUMENT, "null rotary buffer");
    if (!aligned_to_value(a->q, a->in_dtype) || !aligned_to_value(a->k, a->in_dtype) ||
        !aligned_to_value(a->v, a->in_dtype) || !aligned_to_value(a->q_out, a->out_dtype) ||
        !aligned_to_value(a->k_cache, a->out_dtype) || !aligned_to_value(a->v_cache, a->out_dtype))
        return set_error(FM_STATUS_INVALID_ARGUMENT, "rotary buffer is not aligned to its values");
    if (a->tokens > 0x7FFFFFFFu) return set_error(FM_STATUS_SHAPE_MISMATCH, "too many tokens in a call");
    int *status = device_status_word();
    const uint32_t half = a->rot_dim / 2, kvh = cached ? a->kv_heads : 0;
    auto eights = [](int64_t v) { return v % 8 == 0; };
    bool vec = eights(a->head_dim) && eights(a->interleaved ? a->rot_dim : half) && eights(a->q_token_stride) &&
               eights(a->q_head_stride) && eights(a->q_out_token_stride) && eights(a->q_out_head_stride) &&
               aligned16(a->q) && aligned16(a->q_out);
    if (cached)
        vec = vec && eights(a->k_token_stride) && eights(a->k_head_stride) && eights(a->v_token_stride) &&
              eights(a->v_head_stride) && eights(a->cache_page_stride) && eights(a->cache_head_stride) &&
              eights(a->cache_row_stride) && aligned16(a->k) && aligned16(a->v) && aligned16(a->k_cache) &&
              aligned16(a->v_cache);
    const uint32_t unit = vec ? 8 : 1;
    const uint32_t head_items = (a->head_dim - (a->interleaved && vec ? 0 : half)) / unit;
    const uint32_t value_items = a->head_dim / unit;
    const RopeParams p{a->q, a->k, a->v, a->q_out, a->k_cache, a->v_cache, a->positions, a->slots, a->inv_freq,
                       a->q_token_stride, a->q_head_stride, a->k_token_stride, a->k_head_stride, a->v_token_stride,
                       a->v_head_stride, a->q_out_token_stride, a->q_out_head_stride, a->cache_page_stride,
                       a->cache_head_stride, a->cache_row_stride, a->in_dtype, a->out_dtype, a->heads, kvh,
                       a->head_dim, a->rot_dim, a->attention_factor, cached ? a->page_size : 1,
                       cached ? static_cast<uint64_t>(a->n_pages) * a->page_size : 0, head_items, value_items,
                       (a->heads + kvh) * head_items + kvh * value_items, status};
    // few tokens: a token's items over several CTAs, until every SM has one
    const uint32_t rounds = (p.items + ROPE_THREADS - 1) / ROPE_THREADS;
    uint32_t parts = static_cast<uint32_t>(device_sm_count()) / a->tokens;
    parts = parts < 1 ? 1 : parts > rounds ? rounds : parts;
    const uint32_t each = (rounds + parts - 1) / parts;
    uint32_t threads = (p.items + parts * each - 1) / (parts * each);
    threads = (threads + 31) & ~31u;
    const dim3 grid(a->tokens, parts);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (vec && a->interleaved)
        rope_append_kernel<true, true><<<grid, threads, 0, s>>>(p);
    else if (vec)
        rope_append_kernel<true, false><<<grid, threads, 0, s>>>(p);
    else if (a->interleaved)
        rope_append_kernel<false, true><<<grid, threads, 0, s>>>(p);
    else
        rope_append_kernel<false, false><<<grid, threads, 0, s>>>(p);
    return check_launch("rope_append_kernel");
}
