// logprobs.cu -- log probabilities of given tokens, with entropy and the most probable
// alternatives, from the logits of an output head.
//
//   z = scale * logits,  L = log sum_i e^(z_i),  log p_i = z_i - L,  H = -sum_i p_i log p_i
//
// One read of the logits, whatever is asked of them.  Each thread streams chunks of 16
// bytes with a reference value x0 and, over d = x - x0 in units of log2 (t = d scale log2 e),
// the sums of 2^t and of t 2^t, which give L and H; the reference moves only when a value
// exceeds it by 2^8, since any reference in that range gives the same sums.  A difference of
// inputs loses nothing that a product scale * x would lose at large x.
//
// The k most probable values need no second pass either.  A thread keeps the place of its
// largest value.  By (value, lower place) these places are distinct, and whatever belongs to
// the k first of a row lies in one of the k threads whose places come first: every value
// elsewhere is preceded by those k.  So only these threads' chunks, k of hundreds, are read
// again (from L2), and of them what does not come behind the last of the k places is sorted.
//
// A CTA takes a row; where rows are few a cluster does, whose CTAs are joined through
// shared memory.
#include <cfloat>
#include <cmath>
#include <string>

#include "launch.cuh"
#include "ptx.cuh"
#include "vec8.cuh"

namespace fmb {
namespace {

constexpr uint32_t LP_MAX_TOP = 32, LP_LIST = 1024, LP_MAX_CLUSTER = 8;
constexpr float LP_LEAST = -200.0f; // 2^t is 0 from here down; a finite t keeps t 2^t a number

struct LogProbParams {
    const void *logits;
    int64_t stride;
    uint32_t vocab, top;
    const int32_t *tokens;
    float *logprobs, *entropy, *top_logprobs;
    int32_t *top_ids;
    float to_log2; // scale * log2(e)
    double scale;
    int *status;
};

// Larger values have larger codes; NaN is coded as -inf, -0 as 0.  No value has code 0.
__device__ __forceinline__ uint32_t code_of(float x) {
    const uint32_t u = __float_as_uint(x == x ? x + 0.0f : -INFINITY);
    return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t code) {
    return __uint_as_float(code >> 31 ? code & 0x7FFFFFFFu : ~code);
}
// By value, then by lower place: larger keys come first.
__device__ __forceinline__ uint64_t key_of(uint32_t code, uint32_t place) {
    return static_cast<uint64_t>(code) << 32 | static_cast<uint32_t>(~place);
}
__device__ __forceinline__ uint32_t place_of(uint64_t key) { return ~static_cast<uint32_t>(key); }

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

template <int T> constexpr int LP_VEC = 16 / static_cast<int>(x_size(T));

template <int T> __device__ __forceinline__ void unpack16(uint4 w, float (&v)[LP_VEC<T>]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (T == FM_X_F32) {
            v[i] = __uint_as_float(u[i]);
        } else if constexpr (T == FM_X_BF16) {
            v[2 * i] = __uint_as_float(u[i] << 16);
            v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
}

// A row as a ragged head, whole chunks at 16-byte addresses, and a ragged tail.  Chunk i is
// thread i modulo the row's threads's; the head is thread 0's, and the tail is chunk `whole`.
template <int T> struct Row {
    const char *at;
    uint32_t vocab, head, whole;
    __device__ __forceinline__ Row(const LogProbParams &p, uint64_t row) {
        constexpr uint32_t S = x_size(T), V = LP_VEC<T>;
        at = static_cast<const char *>(p.logits) + static_cast<int64_t>(row) * p.stride * S;
        vocab = p.vocab;
        const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(at) & 15u) / S;
        head = off ? V - off : 0;
        if (head > vocab) head = vocab;
        whole = (vocab - head) / V;
    }
    __device__ __forceinline__ uint32_t first_of(uint32_t chunk) const { return head + chunk * LP_VEC<T>; }
    __device__ __forceinline__ uint4 load(uint32_t chunk) const {
        return __ldg(reinterpret_cast<const uint4 *>(at + static_cast<uint64_t>(first_of(chunk)) * x_size(T)));
    }
    // values [first, first + n), n < V; the others -inf
    __device__ __forceinline__ void ragged(uint32_t first, uint32_t n, float (&v)[LP_VEC<T>]) const {
#pragma unroll
        for (int j = 0; j < LP_VEC<T>; ++j) v[j] = static_cast<uint32_t>(j) < n ? load1(at, T, first + j) : -INFINITY;
    }
};

// A thread's sums, and its first place by (value, lower place).
struct Running {
    float ref = -FLT_MAX, sum = 0.0f, tsum = 0.0f;
    float best = -INFINITY;
    uint32_t place = 0xFFFFFFFFu; // the first value's of the chunk that holds it; none yet

    template <int V> __device__ __forceinline__ void add(const float (&v)[V], uint32_t first, float c, float step) {
        float high = v[0];
#pragma unroll
        for (int j = 1; j < V; ++j) high = fmaxf(high, v[j]);
        if (high > best || place == 0xFFFFFFFFu) {
            best = fmaxf(high, -INFINITY);
            place = first;
        }
        if (high > ref + step) {
            const float dt = fmaxf((ref - high) * c, LP_LEAST), f = exp2_approx(dt);
            tsum = f * fmaf(dt, sum, tsum);
            sum *= f;
            ref = high;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float t = max_nan((v[j] - ref) * c, LP_LEAST), e = exp2_approx(t);
            sum += e;
            tsum = fmaf(e, t, tsum);
        }
    }
    // the sums for another reference that is not below this one
    __device__ __forceinline__ void move(float to, float c) {
        const float dt = max_nan((ref - to) * c, LP_LEAST), f = exp2_approx(dt);
        tsum = f * fmaf(dt, sum, tsum);
        sum *= f;
        ref = to;
    }
};

__device__ __forceinline__ uint64_t warp_max_key(uint64_t key) {
    const uint32_t hi = static_cast<uint32_t>(key >> 32), top = __reduce_max_sync(0xFFFFFFFFu, hi);
    const uint32_t lo = __reduce_max_sync(0xFFFFFFFFu, hi == top ? static_cast<uint32_t>(key) : 0u);
    return static_cast<uint64_t>(top) << 32 | lo;
}

// The warp's keys, largest in lane 0.
__device__ __forceinline__ uint64_t warp_sort(uint64_t key, uint32_t lane) {
#pragma unroll
    for (uint32_t size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (uint32_t dist = size / 2; dist > 0; dist >>= 1) {
            const uint64_t other = __shfl_xor_sync(0xFFFFFFFFu, key, dist);
            const bool larger = ((lane & dist) == 0) == ((lane & size) == 0 || size == 32);
            if ((other > key) == larger) key = other;
        }
    return key;
}

struct LPShared {
    uint64_t sorted[32][32]; // the warps' threads by their places
    uint64_t list[LP_LIST];
    uint64_t first[LP_MAX_TOP]; // the row's (the CTA's part's) first values
    uint64_t chosen[LP_MAX_TOP];
    float ref[32], sum[32], tsum[32];
    float all[3]; // ref, sum, tsum of the CTA
    uint32_t n;
};

// The k first of n keys to `first`, by counting for each how many come before it.
__device__ __forceinline__ void rank_keys(const uint64_t *keys, uint32_t n, uint32_t k, uint64_t *first) {
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
        const uint64_t key = keys[i];
        uint32_t before = 0;
        for (uint32_t j = 0; j < n; ++j) before += keys[j] > key;
        if (before < k) first[before] = key;
    }
}

// The k first values of the CTA's part of a row (chunks cta_first.. modulo all), to s.first.
template <int T>
__device__ __forceinline__ void select_top(const Row<T> &row, const Running &mine, uint32_t k, uint32_t rank,
                                           uint32_t threads, LPShared &s) {
    constexpr uint32_t V = LP_VEC<T>;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, warps = blockDim.x / 32;
    uint64_t key = mine.place == 0xFFFFFFFFu ? 0 : key_of(code_of(mine.best), mine.place);
    s.sorted[warp][lane] = warp_sort(key, lane);
    if (threadIdx.x == 0) s.n = 0;
    __syncthreads();
    if (warp == 0) {
        // lane w goes down warp w's list
        uint32_t next = 0;
        uint64_t head = lane < warps ? s.sorted[lane][0] : 0;
        for (uint32_t r = 0; r < k; ++r) {
            const uint64_t top = warp_max_key(head);
            if (lane == 0) s.chosen[r] = top;
            if (head == top) head = ++next < 32 && lane < warps ? s.sorted[lane][next] : 0;
        }
    }
    __syncthreads();
    // what does not come behind the last of them (0: fewer threads than k have a place)
    const uint64_t bound = s.chosen[k - 1];
    const uint32_t bound_code = static_cast<uint32_t>(bound >> 32), bound_place = bound ? place_of(bound) : 0xFFFFFFFFu;
    const uint32_t tail = row.vocab - row.first_of(row.whole);
    const uint32_t rounds = (row.whole + threads - 1) / threads, per = rounds + 2;
    auto visit = [&](auto &&take) {
        for (uint32_t w = threadIdx.x; w < k * per; w += blockDim.x) {
            const uint64_t from = s.chosen[w / per];
            if (!from) continue;
            const uint32_t place = place_of(from), owner = place < row.head ? 0 : (place - row.head) / V % threads;
            const uint32_t i = w % per;
            float v[V];
            uint32_t first = 0, n = 0;
            if (i < rounds) {
                const uint32_t chunk = owner + i * threads;
                if (chunk >= row.whole) continue;
                first = row.first_of(chunk), n = V;
                unpack16<T>(row.load(chunk), v);
            } else {
                if (i == rounds && owner == 0) n = row.head;
                if (i > rounds && owner == row.whole % threads) first = row.first_of(row.whole), n = tail;
                row.ragged(first, n, v);
            }
#pragma unroll
            for (uint32_t j = 0; j < V; ++j) {
                const uint32_t code = code_of(v[j]);
                if (j < n && (code > bound_code || (code == bound_code && first <= bound_place))) take(key_of(code, first + j));
            }
        }
    };
    visit([&](uint64_t key) {
        const uint32_t at = atomicAdd(&s.n, 1u);
        if (at < LP_LIST) s.list[at] = key;
    });
    if (threadIdx.x < k) s.first[threadIdx.x] = 0;
    __syncthreads();
    if (s.n <= LP_LIST) {
        rank_keys(s.list, s.n, k, s.first);
    } else {
        // more than the list holds (values that grow or fall along the row in steps of a thread's): one at a time
        uint64_t last = ~0ull;
        for (uint32_t r = 0; r < k; ++r) {
            uint64_t best = 0;
            visit([&](uint64_t key) {
                if (key < last && key > best) best = key;
            });
            best = warp_max_key(best);
            __syncthreads();
            if (lane == 0) s.list[warp] = best;
            __syncthreads();
            last = 0;
            for (uint32_t w = 0; w < warps; ++w) last = s.list[w] > last ? s.list[w] : last;
            if (threadIdx.x == 0) s.first[r] = last;
        }
    }
    __syncthreads();
}

template <int T>
__global__ void __launch_bounds__(1024) logprobs_kernel(const LogProbParams p, uint32_t ranks) {
    constexpr int V = LP_VEC<T>, U = T == FM_X_F32 ? 4 : 4;
    __shared__ LPShared s;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, warps = blockDim.x / 32;
    const uint32_t rank = blockIdx.x % ranks, threads = blockDim.x * ranks;
    const uint64_t r = blockIdx.x / ranks;
    after_stream();
    let_next();
    const Row<T> row(p, r);
    const uint32_t me = rank * blockDim.x + threadIdx.x;
    const float c = p.to_log2, step = 8.0f / c;
    float chosen = 0.0f;
    int32_t token = -1;
    if (me == 0) {
        token = p.tokens[r];
        if (token >= 0 && static_cast<uint32_t>(token) < row.vocab) chosen = load1(row.at, T, static_cast<uint32_t>(token));
    }
    Running mine;
    float v[V];
    if (me == 0 && row.head) {
        row.ragged(0, row.head, v);
        mine.add(v, 0, c, step);
    }
    uint32_t i = me;
    for (; i + (U - 1) * threads < row.whole; i += U * threads) {
        uint4 w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) w[u] = row.load(i + u * threads);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            unpack16<T>(w[u], v);
            mine.add(v, row.first_of(i + u * threads), c, step);
        }
    }
    for (; i < row.whole; i += threads) {
        unpack16<T>(row.load(i), v);
        mine.add(v, row.first_of(i), c, step);
    }
    const uint32_t tail = row.vocab - row.first_of(row.whole);
    if (tail && me == row.whole % threads) {
        row.ragged(row.first_of(row.whole), tail, v);
        mine.add(v, row.first_of(row.whole), c, step);
    }

    // the CTA's sums
    float top = mine.ref;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    Running all = mine;
    all.move(top, c);
    all.sum = warp_sum(all.sum);
    all.tsum = warp_sum(all.tsum);
    if (lane == 0) {
        s.ref[warp] = top;
        s.sum[warp] = all.sum;
        s.tsum[warp] = all.tsum;
    }
    __syncthreads();
    if (warp == 0) {
        all.ref = lane < warps ? s.ref[lane] : -FLT_MAX;
        all.sum = lane < warps ? s.sum[lane] : 0.0f;
        all.tsum = lane < warps ? s.tsum[lane] : 0.0f;
        top = all.ref;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        all.move(top, c);
        all.sum = warp_sum(all.sum);
        all.tsum = warp_sum(all.tsum);
        if (lane == 0) {
            s.all[0] = top;
            s.all[1] = all.sum;
            s.all[2] = all.tsum;
        }
    }
    if (p.top) select_top<T>(row, mine, p.top, rank, threads, s);
    else __syncthreads();

    if (ranks > 1) {
        cluster_sync();
        if (rank == 0) {
            float ref[LP_MAX_CLUSTER], sum[LP_MAX_CLUSTER], tsum[LP_MAX_CLUSTER];
            top = -FLT_MAX;
#pragma unroll
            for (uint32_t q = 0; q < LP_MAX_CLUSTER; ++q) {
                ref[q] = -FLT_MAX;
                sum[q] = tsum[q] = 0.0f;
                if (q >= ranks) continue;
                ref[q] = cluster_load(smem_u32(&s.all[0]), q);
                sum[q] = cluster_load(smem_u32(&s.all[1]), q);
                tsum[q] = cluster_load(smem_u32(&s.all[2]), q);
            }
            for (uint32_t w = threadIdx.x; w < ranks * p.top; w += blockDim.x)
                s.list[w] = cluster_load64(smem_u32(&s.first[w % p.top]), w / p.top);
#pragma unroll
            for (uint32_t q = 0; q < LP_MAX_CLUSTER; ++q) top = fmaxf(top, ref[q]);
            all.sum = all.tsum = 0.0f;
#pragma unroll
            for (uint32_t q = 0; q < LP_MAX_CLUSTER; ++q) {
                Running part;
                part.ref = ref[q];
                part.sum = sum[q];
                part.tsum = tsum[q];
                part.move(top, c);
                all.sum += part.sum;
                all.tsum += part.tsum;
            }
        }
        cluster_sync(); // nobody leaves, and nothing of rank 0's is overwritten, while it is read
        if (rank != 0) return;
        if (threadIdx.x == 0) {
            s.all[0] = top;
            s.all[1] = all.sum;
            s.all[2] = all.tsum;
        }
        rank_keys(s.list, ranks * p.top, p.top, s.first);
        __syncthreads();
    }
    // sum 0: a row of nothing but -inf
    const float ref = s.all[0], sum = s.all[1];
    const double log_sum = log(static_cast<double>(sum));
    auto log_p = [&](float x) {
        return sum == 0.0f ? -INFINITY : static_cast<float>(p.scale * (static_cast<double>(x) - ref) - log_sum);
    };
    if (threadIdx.x == 0) {
        if (token >= 0 && static_cast<uint32_t>(token) >= row.vocab) {
            raise_device_status(p.status, FM_STATUS_INVALID_ARGUMENT);
            p.logprobs[r] = NAN;
        } else {
            p.logprobs[r] = token < 0 ? 0.0f : log_p(chosen);
        }
        const float h = sum == 0.0f ? 0.0f : static_cast<float>(log_sum - 0.69314718055994531 * s.all[2] / sum);
        p.entropy[r] = h < 0.0f ? 0.0f : h;
    }
    if (threadIdx.x < p.top) {
        const uint64_t key = s.first[threadIdx.x], at = r * p.top + threadIdx.x;
        p.top_logprobs[at] = log_p(value_of(static_cast<uint32_t>(key >> 32)));
        p.top_ids[at] = static_cast<int32_t>(place_of(key));
    }
}

} // namespace
} // namespace fmb

using namespace fmb;

extern "C" int fmcuda_token_logprobs(const fmcuda_token_logprobs_args *a, void *stream) {
    if (!a) return set_error(FM_STATUS_INVALID_ARGUMENT, "null log probability arguments");
    if (!is_float_x(a->dtype)) return set_error(FM_STATUS_INVALID_ARGUMENT, "logits must be float32, bfloat16 or float16");
    if (a->vocab == 0 || a->vocab > (1u << 30)) return set_error(FM_STATUS_SHAPE_MISMATCH, "vocabulary must be 1 to 2^30");
    if (a->top > LP_MAX_TOP || a->top > a->vocab)
        return set_error(FM_STATUS_INVALID_ARGUMENT, "top must be at most 32 and at most the vocabulary");
    if (!(a->scale >= 1e-30 && a->scale <= 1e30))
        return set_error(FM_STATUS_INVALID_ARGUMENT, "scale must be 1e-30 to 1e30");
    if (a->tokens > 0x7FFFFFFFu) return set_error(FM_STATUS_SHAPE_MISMATCH, "too many tokens in a call");
    if (a->tokens > 1 && a->row_stride < static_cast<int64_t>(a->vocab))
        return set_error(FM_STATUS_SHAPE_MISMATCH, "row stride is smaller than the vocabulary");
    if (a->tokens == 0) return FM_STATUS_OK;
    if (!a->logits || !a->token || !a->logprobs || !a->entropy || (a->top && (!a->top_logprobs || !a->top_ids)))
        return set_error(FM_STATUS_INVALID_ARGUMENT, "null log probability buffer");
    if (!aligned_to_value(a->logits, a->dtype) || !aligned_to_value(a->token, FM_X_F32) ||
        !aligned_to_value(a->logprobs, FM_X_F32) || !aligned_to_value(a->entropy, FM_X_F32) ||
        (a->top && (!aligned_to_value(a->top_logprobs, FM_X_F32) || !aligned_to_value(a->top_ids, FM_X_F32))))
        return set_error(FM_STATUS_INVALID_ARGUMENT, "log probability buffer is not aligned to its values");
    const LogProbParams p{a->logits,       a->row_stride,   a->vocab,
                          a->top,          a->token,        a->logprobs,
                          a->entropy,      a->top_logprobs, a->top_ids,
                          static_cast<float>(a->scale * 1.4426950408889634), a->scale, device_status_word()};
    // threads with a few chunks each; rows that leave SMs idle go to clusters
    const uint64_t chunks = static_cast<uint64_t>(a->vocab) * x_size(a->dtype) / 16;
    const uint64_t sms = static_cast<uint64_t>(device_sm_count());
    uint32_t ranks = 1, threads = 32;
    while (ranks < LP_MAX_CLUSTER && a->tokens * ranks * 2 <= sms && chunks >= ranks * 2048ull) ranks *= 2;
    while (threads < 512 && chunks > static_cast<uint64_t>(threads) * ranks * 8) threads *= 2;
    const Launch l{dim3(a->tokens * ranks), threads, 0, ranks};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a->dtype == FM_X_F32) return launch("logprobs_kernel", logprobs_kernel<FM_X_F32>, l, s, p, ranks);
    if (a->dtype == FM_X_BF16) return launch("logprobs_kernel", logprobs_kernel<FM_X_BF16>, l, s, p, ranks);
    return launch("logprobs_kernel", logprobs_kernel<FM_X_F16>, l, s, p, ranks);
}
