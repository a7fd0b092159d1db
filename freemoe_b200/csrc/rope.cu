// rope.cu -- rotary positions of new queries and keys, and the write of new
// keys and values into the pages of a cache.
//
//   (a, b) -> (a cos t - b sin t, a sin t + b cos t),  t = position * inv_freq[i]
//
// (src/rope.cpp of the reference turns one head at a time on the host).  The
// operator is one read of q, k and v and one write of q and of two cache rows a
// token; the cosines of a token are shared by all of its heads.  A CTA takes a
// few tokens, whose cosines its threads work out together before the barrier, or
// a part of one token's heads when there are too few tokens to fill the GPU.
//
// The angle of a far position does not fit f32 (at position 2^17 its last bit
// is 2^-7 radians), so the product is taken in turns in 64 bits, its whole part
// dropped, and only the fraction of a turn goes to f32: three 64-bit operations
// a pair, once for all heads.
#include <cmath>
#include <string>

#include "launch.cuh"
#include "vec8.cuh"

namespace fmb {
namespace {

constexpr uint32_t ROPE_THREADS = 256;
constexpr uint32_t ROPE_MAX_DIM = 1024, ROPE_TURNS = ROPE_MAX_DIM / 2, ROPE_BATCH = 8;

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
    uint32_t head_items, value_items; // eights (or pairs of eights) of a rotated head, of a value head
    uint32_t tokens, batch;                  // tokens a CTA takes together
    int *status;
};

// The cosines of the CTA's tokens, and their rows of the cache (-1: a slot below zero or,
// reported, past the cache); ends with the CTA's barrier.
__device__ __forceinline__ void rope_tokens(const RopeParams &p, uint32_t t0, uint32_t n, float2 *s_turns,
                                            int64_t *s_row) {
    const uint32_t half = p.rot / 2;
    for (uint32_t i = threadIdx.x; i < n * half; i += blockDim.x) {
        const uint32_t k = i / half;
        const double turns = static_cast<double>(p.positions[t0 + k]) *
                             static_cast<double>(p.inv_freq[i - k * half]) * 0.15915494309189533577; // 1 / (2 pi)
        float sn, cs;
        sincospif(2.0f * static_cast<float>(turns - rint(turns)), &sn, &cs);
        s_turns[i] = make_float2(cs * p.factor, sn * p.factor);
    }
    if (threadIdx.x < n) {
        int64_t row = -1;
        if (p.kc) {
            const int64_t slot = p.slots[t0 + threadIdx.x];
            if (slot >= 0 && static_cast<uint64_t>(slot) < p.n_slots) {
                const int64_t page = slot / p.page_size;
                row = page * p.cp + (slot - page * p.page_size) * p.cr;
            } else if (slot >= 0 && blockIdx.y == 0) {
                raise_device_status(p.status, FM_STATUS_INVALID_ARGUMENT);
            }
        }
        s_row[threadIdx.x] = row;
    }
    __syncthreads();
}

// Eight values of a compile-time type.
template <int T> __device__ __forceinline__ Raw8 rope_load(const char *src) {
    Raw8 r;
    r.a = r.b = *reinterpret_cast<const uint4 *>(src);
    if constexpr (T == FM_X_F32) r.b = reinterpret_cast<const uint4 *>(src)[1];
    return r;
}

__device__ __forceinline__ uint4 rope_shuffle(uint4 v, uint32_t lane) {
    return make_uint4(__shfl_sync(0xFFFFFFFFu, v.x, lane), __shfl_sync(0xFFFFFFFFu, v.y, lane),
                      __shfl_sync(0xFFFFFFFFu, v.z, lane), __shfl_sync(0xFFFFFFFFu, v.w, lane));
}

// Heads, strides and (not interleaved) rot/2 in whole eights.  A thread keeps its place
// in the head -- eight values; PAIRED: eight pairs (i, i + rot/2) -- and up to U of the
// heads of q, k and (not PAIRED, where their places are the same) v, whose addresses only
// move on from token to token of the CTA's batch: per token U loads under way together,
// then the turns and the stores.  HALVES: the partners at i +- rot/2 come from the lane
// that loaded them, where a head's eights divide a warp; PAIRED is for heads that do not.
// Measured with 8192 tokens of 32 + 8 heads of 128, bf16, interleaved (201 MB, 31 us at the
// measured copy rate): 37 us; U = 2 or 4, 39; an index over all of a token's eights with its
// divisions, 44 (issue slots 65% busy); the cosines worked out by every thread for
// itself, 64.  Bound by the loads under way: registers against warps.  HALVES: 42 us, from
// f32 to bf16 (302 MB) 65 against 47; it reads twice the cosines for an eight and shuffles,
// and what bounds it has not been profiled.
enum { ROPE_INTER, ROPE_HALVES, ROPE_PAIRED };

template <int LAYOUT, int IN, int OUT>
__global__ void __launch_bounds__(ROPE_THREADS, LAYOUT == ROPE_PAIRED && IN == FM_X_F32 ? 2 : 4)
    rope_append_kernel(const RopeParams p) {
    constexpr bool INTER = LAYOUT == ROPE_INTER, PAIRED = LAYOUT == ROPE_PAIRED;
    constexpr int PAIRS = INTER ? 4 : 8, U = IN == FM_X_F32 || PAIRED ? 2 : 3;
    constexpr int SI = x_size(IN), SO = x_size(OUT);
    __shared__ float2 s_turns[ROPE_TURNS];
    __shared__ int64_t s_row[ROPE_BATCH];
    const uint32_t t0 = blockIdx.x * p.batch, n = p.tokens - t0 < p.batch ? p.tokens - t0 : p.batch;
    const uint32_t half = p.rot / 2, at_once = blockDim.x / p.head_items; // heads at once
    const uint32_t item = threadIdx.x % p.head_items, lane_head = threadIdx.x / p.head_items;
    const bool pair = item * 8 < (PAIRED ? half : p.rot);
    const uint32_t ea = item * 8 + (!PAIRED || pair ? 0 : half); // copied values lie behind the pairs
    const uint32_t step = at_once * gridDim.y, turned = p.heads + p.kv_heads;
    const uint32_t heads = lane_head >= at_once ? 0 : PAIRED ? turned : turned + p.kv_heads;
    // HALVES: the lane with the partners, and whether they are the first of their pairs
    const bool second = item * 8 >= half;
    const uint32_t partner = (threadIdx.x & 31u) + (pair ? second ? 0u - half / 8 : half / 8 : 0u);
    const float2 *my_turns = s_turns + (INTER ? item * 4 : LAYOUT == ROPE_HALVES && second ? ea - half : ea);
    after_stream();
    let_next();
    bool ready = false;
    uint32_t h1 = blockIdx.y * at_once + lane_head;
    // whole warps go round together: lanes exchange inside
    while (__any_sync(0xFFFFFFFFu, h1 < heads || !ready)) {
        const char *src[U];
        char *dst[U];
        int64_t move[U];
        bool here[U], cached[U], turns[U];
#pragma unroll
        for (int x = 0; x < U; ++x) {
            const uint32_t h = h1 + x * step;
            here[x] = h < heads;
            cached[x] = h >= p.heads;
            turns[x] = pair && h < turned;
            const bool key = h < turned;
            if (!cached[x]) {
                src[x] = static_cast<const char *>(p.q) + (static_cast<int64_t>(t0) * p.qt + h * p.qh + ea) * SI;
                dst[x] = static_cast<char *>(p.q_out) + (static_cast<int64_t>(t0) * p.ot + h * p.oh + ea) * SO;
                move[x] = p.qt * SI;
            } else {
                const uint32_t c = h - (key ? p.heads : turned);
                const int64_t from = static_cast<int64_t>(t0) * (key ? p.kt : p.vt) + c * (key ? p.kh : p.vh);
                src[x] = static_cast<const char *>(key ? p.k : p.v) + (from + ea) * SI;
                dst[x] = static_cast<char *>(key ? p.kc : p.vc) + (c * p.ch + ea) * SO;
                move[x] = (key ? p.kt : p.vt) * SI;
            }
        }
        Raw8 a[U], b[PAIRED ? U : 1];
        auto load = [&] {
#pragma unroll
            for (int x = 0; x < U; ++x) {
                if (here[x]) {
                    a[x] = rope_load<IN>(src[x]);
                    if (PAIRED && turns[x]) b[x] = rope_load<IN>(src[x] + half * SI);
                }
                src[x] += move[x];
            }
        };
        load();
        if (!ready) rope_tokens(p, t0, n, s_turns, s_row); // every thread's first round: its barrier
        ready = true;
#pragma unroll 1
        for (uint32_t k = 0; k < n; ++k) {
            if (k) load();
            const int64_t row = s_row[k];
            float2 cs[PAIRS];
            if (pair) {
#pragma unroll
                for (int j = 0; j < PAIRS; ++j)
                    if (!INTER || item * 4 + j < half) cs[j] = my_turns[k * half + j];
            }
#pragma unroll
            for (int x = 0; x < U; ++x) {
                float f[8], g[8];
                Raw8 other;
                if constexpr (LAYOUT == ROPE_HALVES) {
                    other.a = rope_shuffle(a[x].a, partner);
                    other.b = IN == FM_X_F32 ? rope_shuffle(a[x].b, partner) : other.a;
                }
                if (!here[x] || (cached[x] && row < 0)) continue;
                char *to = dst[x] + (cached[x] ? row : k * p.ot) * SO;
                raw8_unpack(a[x], IN, f);
                if (!turns[x]) {
                    store8(to, OUT, 0, f);
                } else if (INTER) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const bool in = item * 4 + j < half; // the last eight's other values are copied
                        g[2 * j] = in ? f[2 * j] * cs[j].x - f[2 * j + 1] * cs[j].y : f[2 * j];
                        g[2 * j + 1] = in ? f[2 * j] * cs[j].y + f[2 * j + 1] * cs[j].x : f[2 * j + 1];
                    }
                    store8(to, OUT, 0, g);
                } else if (LAYOUT == ROPE_HALVES) {
                    raw8_unpack(other, IN, g);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float sn = second ? cs[j % PAIRS].y : -cs[j % PAIRS].y;
                        f[j] = f[j] * cs[j % PAIRS].x + g[j] * sn;
                    }
                    store8(to, OUT, 0, f);
                } else {
                    raw8_unpack(b[PAIRED ? x : 0], IN, g);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float c = f[j] * cs[j % PAIRS].x - g[j] * cs[j % PAIRS].y;
                        g[j] = f[j] * cs[j % PAIRS].y + g[j] * cs[j % PAIRS].x;
                        f[j] = c;
                    }
                    store8(to, OUT, 0, f);
                    store8(to + half * SO, OUT, 0, g);
                }
            }
        }
        h1 += U * step;
    }
    if (!PAIRED) return;
    // values: copied, eight at a time, all tokens of the batch
    const uint32_t all = p.kv_heads * p.value_items;
    for (uint32_t i = blockIdx.y * blockDim.x + threadIdx.x; i < all; i += gridDim.y * blockDim.x) {
        const uint32_t h = i / p.value_items, e = i % p.value_items * 8;
        const char *src =
            static_cast<const char *>(p.v) + (static_cast<int64_t>(t0) * p.vt + h * p.vh + e) * SI;
        char *dst = static_cast<char *>(p.vc) + (h * p.ch + e) * SO;
#pragma unroll 4
        for (uint32_t k = 0; k < n; ++k) {
            const int64_t row = s_row[k];
            if (row < 0) continue;
            float f[8];
            raw8_unpack(rope_load<IN>(src + k * p.vt * SI), IN, f);
            store8(dst + row * SO, OUT, 0, f);
        }
    }
}

// Any widths, strides and alignments: an item is one pair or one value, consecutive
// threads take consecutive ones.  (Four items of a thread under way together: 24 us, not 17,
// for 2164 tokens of 17 heads of 128, 126 of them turned.)
template <bool INTER> __global__ void __launch_bounds__(ROPE_THREADS) rope_append_any_kernel(const RopeParams p) {
    __shared__ float2 s_turns[ROPE_TURNS];
    __shared__ int64_t s_row[ROPE_BATCH];
    const int64_t t = blockIdx.x;
    after_stream();
    let_next();
    rope_tokens(p, blockIdx.x, 1, s_turns, s_row);
    const int64_t cache_row = s_row[0];
    const uint32_t half = p.rot / 2, turned = p.heads + p.kv_heads, head_items = p.dim - half;
    const uint32_t items = turned * head_items + p.kv_heads * p.dim;
    for (uint32_t it = blockIdx.y * blockDim.x + threadIdx.x; it < items; it += gridDim.y * blockDim.x) {
        const bool turns = it < turned * head_items;
        const uint32_t rest = turns ? it : it - turned * head_items, width = turns ? head_items : p.dim;
        uint32_t h = rest / width;
        const uint32_t item = rest - h * width;
        const void *src = p.q;
        void *dst = p.q_out;
        int64_t from = t * p.qt + h * p.qh, to = t * p.ot + h * p.oh;
        if (!turns || h >= p.heads) {
            if (cache_row < 0) continue;
            if (turns) h -= p.heads;
            src = turns ? p.k : p.v;
            dst = turns ? p.kc : p.vc;
            from = turns ? t * p.kt + h * p.kh : t * p.vt + h * p.vh;
            to = cache_row + h * p.ch;
        }
        if (turns && item < half) {
            const uint32_t ea = INTER ? 2 * item : item, eb = INTER ? ea + 1 : ea + half;
            const float a = load1(src, p.in_t, from + ea), b = load1(src, p.in_t, from + eb);
            const float2 cs = s_turns[item];
            store1(dst, p.out_t, to + ea, a * cs.x - b * cs.y);
            store1(dst, p.out_t, to + eb, a * cs.y + b * cs.x);
        } else {
            const uint32_t e = turns ? item + half : item;
            store1(dst, p.out_t, to + e, load1(src, p.in_t, from + e));
        }
    }
}

template <int LAYOUT, int IN> int launch_rope_in(const RopeParams &p, const Launch &l, cudaStream_t s) {
    auto kfn = p.out_t == FM_X_F32    ? rope_append_kernel<LAYOUT, IN, FM_X_F32>
               : p.out_t == FM_X_BF16 ? rope_append_kernel<LAYOUT, IN, FM_X_BF16>
                                      : rope_append_kernel<LAYOUT, IN, FM_X_F16>;
    return launch("rope_append_kernel", kfn, l, s, p);
}

template <int LAYOUT> int launch_rope(const RopeParams &p, const Launch &l, cudaStream_t s) {
    if (p.in_t == FM_X_F32) return launch_rope_in<LAYOUT, FM_X_F32>(p, l, s);
    if (p.in_t == FM_X_BF16) return launch_rope_in<LAYOUT, FM_X_BF16>(p, l, s);
    return launch_rope_in<LAYOUT, FM_X_F16>(p, l, s);
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
    if (cached && (a->kv_heads == 0 || a->page_size == 0))
        return set_error(FM_STATUS_SHAPE_MISMATCH, "a cache has at least one head and one row a page");
    if (a->tokens == 0) return FM_STATUS_OK; // its k, v and slots may be null beside caches that are not
    if (cached && (!a->k || !a->v || !a->k_cache || !a->v_cache || !a->slots))
        return set_error(FM_STATUS_INVALID_ARGUMENT, "k, v, their caches and slots come together");
    if (!a->q || !a->q_out || !a->positions || (a->rot_dim && !a->inv_freq))
        return set_error(FM_STATUS_INVALID_ARGUMENT, "null rotary buffer");
    if (!aligned_to_value(a->q, a->in_dtype) || !aligned_to_value(a->k, a->in_dtype) ||
        !aligned_to_value(a->v, a->in_dtype) || !aligned_to_value(a->q_out, a->out_dtype) ||
        !aligned_to_value(a->k_cache, a->out_dtype) || !aligned_to_value(a->v_cache, a->out_dtype))
        return set_error(FM_STATUS_INVALID_ARGUMENT, "rotary buffer is not aligned to its values");
    if (reinterpret_cast<uintptr_t>(a->positions) % 4 || (cached && reinterpret_cast<uintptr_t>(a->slots) % 8) ||
        reinterpret_cast<uintptr_t>(a->inv_freq) % 4)
        return set_error(FM_STATUS_INVALID_ARGUMENT, "positions, slots or frequencies are not aligned to their values");
    if (a->tokens > 0x7FFFFFFFu) return set_error(FM_STATUS_SHAPE_MISMATCH, "too many tokens in a call");
    int *status = device_status_word();
    const uint32_t half = a->rot_dim / 2, kvh = cached ? a->kv_heads : 0;
    auto eights = [](int64_t v) { return v % 8 == 0; };
    bool vec = eights(a->head_dim) && (a->interleaved || eights(half)) && eights(a->q_token_stride) &&
               eights(a->q_head_stride) && eights(a->q_out_token_stride) && eights(a->q_out_head_stride) &&
               aligned16(a->q) && aligned16(a->q_out);
    if (cached)
        vec = vec && eights(a->k_token_stride) && eights(a->k_head_stride) && eights(a->v_token_stride) &&
              eights(a->v_head_stride) && eights(a->cache_page_stride) && eights(a->cache_head_stride) &&
              eights(a->cache_row_stride) && aligned16(a->k) && aligned16(a->v) && aligned16(a->k_cache) &&
              aligned16(a->v_cache);
    RopeParams p{a->q, a->k, a->v, a->q_out, a->k_cache, a->v_cache, a->positions, a->slots, a->inv_freq,
                       a->q_token_stride, a->q_head_stride, a->k_token_stride, a->k_head_stride, a->v_token_stride,
                       a->v_head_stride, a->q_out_token_stride, a->q_out_head_stride, a->cache_page_stride,
                       a->cache_head_stride, a->cache_row_stride, a->in_dtype, a->out_dtype, a->heads, kvh,
                       a->head_dim, a->rot_dim, a->attention_factor, cached ? a->page_size : 1,
                       cached ? static_cast<uint64_t>(a->n_pages) * a->page_size : 0,
                       a->head_dim / 8, a->head_dim / 8, a->tokens, 1, status};
    // a head's eights divide a warp: partners are in the same one
    const bool paired = vec && !a->interleaved && half && 256 % a->head_dim;
    if (paired) p.head_items -= half / 8;
    const uint32_t sms = static_cast<uint32_t>(device_sm_count());
    // few tokens: a token's heads (or items) over several CTAs, until every SM has one
    uint32_t threads = ROPE_THREADS, rounds;
    if (vec) {
        const uint32_t at_once = ROPE_THREADS / p.head_items, all = a->heads + kvh * (paired ? 1 : 2);
        rounds = (all + at_once - 1) / at_once;
        if (rounds == 1) threads = (all * p.head_items + 31) & ~31u;
    } else {
        const uint64_t items = static_cast<uint64_t>(a->heads + kvh) * (a->head_dim - half) + kvh * a->head_dim;
        rounds = static_cast<uint32_t>((items + ROPE_THREADS - 1) / ROPE_THREADS);
    }
    uint32_t parts = sms / a->tokens;
    parts = parts < 1 ? 1 : parts > rounds ? rounds : parts;
    if (vec && a->tokens > sms * 4) {
        // more than the GPU holds at once: several to a CTA, as many as its threads have
        // cosines to work out
        const uint32_t most = half ? ROPE_THREADS / half : ROPE_BATCH;
        p.batch = (a->tokens + sms * 4 - 1) / (sms * 4);
        p.batch = p.batch > most ? most : p.batch;
        p.batch = p.batch < 1 ? 1 : p.batch > ROPE_BATCH ? ROPE_BATCH : p.batch;
    }
    const Launch l{dim3((a->tokens + p.batch - 1) / p.batch, parts), threads, 0, 1};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (!vec && a->interleaved) return launch("rope_append_any_kernel", rope_append_any_kernel<true>, l, s, p);
    if (!vec) return launch("rope_append_any_kernel", rope_append_any_kernel<false>, l, s, p);
    if (a->interleaved) return launch_rope<ROPE_INTER>(p, l, s);
    return paired ? launch_rope<ROPE_PAIRED>(p, l, s) : launch_rope<ROPE_HALVES>(p, l, s);
}
