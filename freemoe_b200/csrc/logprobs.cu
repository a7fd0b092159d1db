// logprobs.cu -- log probabilities of given tokens, with entropy and the most probable
// alternatives, from the logits of an output head.
//
//   z = scale * logits,  L = log sum_i e^(z_i),  log p_i = z_i - L,  H = -sum_i p_i log p_i
//
// One read of the logits, whatever is asked of them.  Each thread streams chunks of 32
// bytes with a reference x0 and, over t = (x - x0) scale log2 e, the sums of 2^t and of
// t 2^t, which give L and H; the reference moves only when a value exceeds it by 2^8, since
// any in that range gives the same sums.  A difference of inputs loses nothing that a
// product scale x would lose at large x, and is 0 at x0 itself: a sure token has log
// probability 0.  16-bit logits arrive at ten values a clock and SM, with a dozen issue slots
// for each, so that what is not arithmetic is done for two values or for a chunk at a time;
// -inf (tokens ruled out) is raised to a value whose 2^t is 0, and not looked at again.
// Where no such value is (references or scales at the ends of their range) a chunk goes the
// long way, value by value.
//
// The k most probable values need no second pass either.  A thread keeps its best chunk, by
// its largest value and then by the lower place, and the largest value of its other chunks.
// The threads make 32 or 64 groups; the k-th of the groups' best chunks is a bound that k
// chunks reach, so that nothing that comes behind it belongs to the k first of the row.  A
// thread whose best chunk reaches it reads that chunk again (from L2); the few of which
// another one does as well have all of their chunks read again, by the whole CTA.  What
// these hold up to the bound, little more than k values, is sorted.  (With all chunks of
// every such thread read again, 4096 rows of 128256 in bf16 took 272 us for 32 of them, where
// they take 179 for none.)
//
// A CTA takes a row; where rows are few a cluster does, whose CTAs send their sums and first
// values to one of them.
//
// Measured: 4096 rows of 128256, bf16, 5 alternatives (1.05 GB) 193 to 240 us by machine and
// heat, 67 to 83% of the rate of a copy (exponentials 60% busy, issue slots 65%); without
// alternatives 180 to 205; 2048 rows in f32 171 to 184.  333 rows of 32003, f16, 32 alternatives,
// half of them ruled out 15 us, of which the selection is 4, and 18 with none ruled out; one row of
// 151936 in f32, 20 alternatives, 8.4 us, latency.
#include <cfloat>
#include <cmath>
#include <string>

#include "launch.cuh"
#include "ptx.cuh"
#include "vec8.cuh"

namespace fmb {
namespace {

constexpr uint32_t LP_MAX_TOP = 32, LP_GROUPS = 64, LP_LIST = 1024, LP_MAX_CLUSTER = 8, LP_THREADS = 512, LP_MANY = 256;
constexpr float LP_LEAST = -200.0f; // 2^t is 0 from here down; a finite t keeps t 2^t a number

struct LogProbParams {
    const void *logits;
    int64_t stride;
    uint32_t vocab, top;
    const int32_t *tokens;
    float *logprobs, *entropy, *top_logprobs;
    int32_t *top_ids;
    float c;        // scale * log2(e)
    float raised;   // what values below it are raised to, in the logits' type
    float step;     // values that exceed a reference by it move it: 8 / c
    float nothing;  // a reference over which a chunk of raised values adds nothing
    float ordinary; // a reference from here to -raised goes the short way
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

template <int T> constexpr int LP_VEC = 32 / static_cast<int>(x_size(T)); // values a chunk

struct Chunk {
    uint32_t w[8];
};
// (Not by read-only loads, here and below: the kernel begins while the one that writes the logits may still run.)
__device__ __forceinline__ Chunk load_chunk32(const void *at) {
    Chunk r;
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n"
                 : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]), "=r"(r.w[4]), "=r"(r.w[5]), "=r"(r.w[6]),
                   "=r"(r.w[7])
                 : "l"(at));
    return r;
}

// The same for a chunk that is read a second time, of which single values are looked at again: kept in L1.
__device__ __forceinline__ Chunk load_chunk32_again(const void *at) {
    const uint4 a = *static_cast<const uint4 *>(at), b = static_cast<const uint4 *>(at)[1];
    return Chunk{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
}

// The two values of a 4-byte word.
template <int T> __device__ __forceinline__ float2 two_of(uint32_t u) {
    if constexpr (T == FM_X_BF16) return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
    return __half22float2(*reinterpret_cast<const __half2 *>(&u));
}
template <int T> __device__ __forceinline__ void unpack(const Chunk &x, float (&v)[LP_VEC<T>]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (T == FM_X_F32) {
            v[i] = __uint_as_float(x.w[i]);
        } else {
            const float2 f = two_of<T>(x.w[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
}

// The larger of two values of f32, or of two pairs of 16-bit ones; NaN left out, or kept.
template <int T, bool NAN_KEPT = false> __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    uint32_t r;
    if constexpr (T == FM_X_F32) {
        if constexpr (NAN_KEPT)
            asm("max.NaN.f32 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
        else
            asm("max.f32 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
    } else if constexpr (T == FM_X_BF16) {
        if constexpr (NAN_KEPT)
            asm("max.NaN.bf16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
        else
            asm("max.bf16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
    } else {
        if constexpr (NAN_KEPT)
            asm("max.NaN.f16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
        else
            asm("max.f16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
    }
    return r;
}

// A chunk's largest value, NaN left out.
template <int T> __device__ __forceinline__ float largest(const Chunk &x) {
    const uint32_t a = larger<T>(larger<T>(x.w[0], x.w[1]), larger<T>(x.w[2], x.w[3]));
    const uint32_t b = larger<T>(larger<T>(x.w[4], x.w[5]), larger<T>(x.w[6], x.w[7]));
    const uint32_t top = larger<T>(a, b);
    if constexpr (T == FM_X_F32) return __uint_as_float(top);
    const float2 f = two_of<T>(top);
    return fmaxf(f.x, f.y);
}

// A row as a ragged head, whole chunks at 32-byte addresses, and a ragged tail: chunks 0, 1 ..
// whole and whole + 1, either end of which may be empty.  Chunk i is thread i modulo the row's
// threads's.
template <int T> struct Row {
    const char *at;
    uint32_t vocab, head, whole, tail;
    __device__ __forceinline__ Row(const LogProbParams &p, uint64_t row) {
        constexpr uint32_t S = x_size(T), V = LP_VEC<T>;
        at = static_cast<const char *>(p.logits) + static_cast<int64_t>(row) * p.stride * S;
        vocab = p.vocab;
        const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(at) & 31u) / S;
        head = off ? V - off : 0;
        if (head > vocab) head = vocab;
        whole = (vocab - head) / V;
        tail = vocab - head - whole * V;
    }
    __device__ __forceinline__ uint32_t first_of(uint32_t chunk) const {
        return chunk ? head + (chunk - 1) * LP_VEC<T> : 0;
    }
    __device__ __forceinline__ uint32_t size_of(uint32_t chunk) const {
        return chunk == 0 ? head : chunk <= whole ? LP_VEC<T> : chunk == whole + 1 ? tail : 0;
    }
    // whole chunk i, from 0
    __device__ __forceinline__ const char *whole_at(uint32_t i) const {
        return at + static_cast<uint64_t>(head) * x_size(T) + static_cast<uint64_t>(i) * 32;
    }
    // A chunk at an end, or behind the last; what it lacks is -inf.
    __device__ __noinline__ Chunk end(uint32_t chunk) const {
        const uint32_t first = first_of(chunk), n = size_of(chunk);
        constexpr uint32_t NONE = T == FM_X_F32 ? 0xFF800000u : T == FM_X_BF16 ? 0xFF80FF80u : 0xFC00FC00u;
        Chunk x;
        if (n == 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x.w[i] = NONE;
            return x;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) x.w[i] = 0;
#pragma unroll
        for (uint32_t j = 0; j < LP_VEC<T>; ++j) {
            if constexpr (T == FM_X_F32) {
                x.w[j] = j < n ? reinterpret_cast<const uint32_t *>(at)[first + j] : NONE;
            } else {
                x.w[j / 2] |= (j < n ? reinterpret_cast<const uint16_t *>(at)[first + j] : NONE & 0xFFFFu) << (j % 2 * 16);
            }
        }
        return x;
    }
};

// Sums over the reference `ref`: a value of the row; -FLT_MAX where there are none.
struct Sums {
    float ref = -FLT_MAX, sum = 0.0f, tsum = 0.0f;
    // the same for another reference that is not below
    __device__ __forceinline__ void move(float to, float c) {
        const float dt = max_nan((ref - to) * c, LP_LEAST), f = exp2_approx(dt);
        tsum = f * fmaf(dt, sum, tsum);
        sum *= f;
        ref = to;
    }
};

// A chunk's sums the long way.
template <int T> __device__ __noinline__ float2 long_way(Chunk x, float ref, float c) {
    float v[LP_VEC<T>];
    unpack<T>(x, v);
    float2 r = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int j = 0; j < LP_VEC<T>; ++j) {
        const float t = max_nan((v[j] - ref) * c, LP_LEAST), e = exp2_approx(t);
        r.x += e;
        r.y = fmaf(e, t, r.y);
    }
    return r;
}

// The same while a row goes by, and the thread's best chunk.  Two sums each, for the operations
// that take two values.
template <int T> struct Stream {
    float ref, limit; // a value above the limit moves the reference
    float best, second; // the best chunk's largest value, and the other chunks'
    uint32_t chunk;     // 0xFFFFFFFF: none
    uint64_t sum, tsum;
    float base; // the reference, or where a chunk of the short way is all -inf a value that is high enough
    uint32_t raised;

    // `first`: the thread's first chunk, if there is one
    __device__ __forceinline__ Stream(const LogProbParams &p, uint32_t first)
        : ref(-FLT_MAX), limit(-INFINITY), best(-INFINITY), second(-INFINITY), chunk(first), sum(0), tsum(0), base(p.nothing) {
        if constexpr (T == FM_X_F32)
            raised = __float_as_uint(p.raised);
        else
            raised = pack2(p.raised, p.raised, T);
    }

    // Whole warps come here together, each lane with a chunk of its own.
    __device__ __forceinline__ void add(const LogProbParams &p, Chunk &x, uint32_t at) {
        const float high = largest<T>(x);
        if (high > best) chunk = at;
        second = fmaxf(second, fminf(best, high));
        best = fmaxf(best, high);
        if (__any_sync(0xFFFFFFFFu, high > limit)) move(p, x, high);
        const uint64_t c2 = pack_f32x2(p.c, p.c), to = pack_f32x2(-base, -base);
#pragma unroll
        for (int i = 0; i < 8; ++i) x.w[i] = larger<T, true>(x.w[i], raised);
        float v[LP_VEC<T>];
        unpack<T>(x, v);
#pragma unroll
        for (int j = 0; j < LP_VEC<T>; j += 2) {
            const uint64_t t = mul_f32x2(add_f32x2(pack_f32x2(v[j], v[j + 1]), to), c2);
            float a, b;
            unpack_f32x2(t, a, b);
            const uint64_t e = pack_f32x2(exp2_approx(a), exp2_approx(b));
            sum = add_f32x2(sum, e);
            tsum = fma_f32x2(e, t, tsum);
        }
    }

    // Moves the lanes' references up to their chunks' largest values; a chunk whose reference
    // does not go the short way is added here, and leaves nothing to add.
    __device__ __forceinline__ void move(const LogProbParams &p, Chunk &x, float high) {
        const bool over = high > limit;
        const float to = over && high > ref ? high : ref;
        const float dt = ref == to ? 0.0f : max_nan((ref - to) * p.c, LP_LEAST), f = exp2_approx(dt);
        const uint64_t f2 = pack_f32x2(f, f);
        tsum = mul_f32x2(f2, fma_f32x2(pack_f32x2(dt, dt), sum, tsum));
        sum = mul_f32x2(f2, sum);
        ref = to;
        const bool ordinary = ref >= p.ordinary && ref <= -p.raised;
        base = ordinary ? ref : p.nothing;
        limit = ordinary ? ref + p.step : -INFINITY;
        if (over && !ordinary) {
            const float2 more = long_way<T>(x, ref, p.c);
            sum = add_f32x2(sum, pack_f32x2(more.x, 0.0f));
            tsum = add_f32x2(tsum, pack_f32x2(more.y, 0.0f));
#pragma unroll
            for (int i = 0; i < 8; ++i) x.w[i] = raised;
        }
    }

    __device__ __forceinline__ Sums sums() const {
        Sums r;
        float a, b;
        unpack_f32x2(sum, a, b);
        r.sum = a + b;
        unpack_f32x2(tsum, a, b);
        r.tsum = a + b;
        r.ref = ref;
        return r;
    }
};

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    return v;
}

__device__ __forceinline__ uint64_t warp_max_key(uint64_t key) {
    const uint32_t hi = static_cast<uint32_t>(key >> 32), top = __reduce_max_sync(0xFFFFFFFFu, hi);
    const uint32_t lo = __reduce_max_sync(0xFFFFFFFFu, hi == top ? static_cast<uint32_t>(key) : 0u);
    return static_cast<uint64_t>(top) << 32 | lo;
}

struct LPShared {
    uint64_t groups[LP_GROUPS]; // their best chunks
    uint64_t bound;
    uint64_t list[LP_LIST];
    uint64_t first[LP_MAX_TOP]; // the first values of the row, or of the CTA's part of it
    float ref[LP_THREADS / 32], sum[LP_THREADS / 32], tsum[LP_THREADS / 32];
    // what the cluster's CTAs send to the first one: their first values and their sums
    uint64_t sent[LP_MAX_CLUSTER][LP_MAX_TOP];
    uint32_t before[LP_MAX_CLUSTER][LP_MAX_TOP];
    float sent_sums[3][LP_MAX_CLUSTER];
    uint32_t n, singles, columns;
    uint32_t single[LP_THREADS];  // chunks that are read again
    uint16_t column[LP_THREADS];  // threads whose chunks are all read again
};

// The k first of n keys to `first`, by counting for each how many come before it.
__device__ __forceinline__ void rank_keys(const uint64_t *keys, uint32_t n, uint32_t k, uint64_t *first) {
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
        const uint64_t key = keys[i];
        uint32_t before = 0;
#pragma unroll 8
        for (uint32_t j = 0; j < n; ++j) before += keys[j] > key;
        if (before < k) first[before] = key;
    }
}

// The k first of the keys that the cluster's CTAs have sent, 32 places each, each in order (0: no more):
// a key's place is its own in its list and what comes before it in the others.  A warp takes a list,
// or half of what it is compared with, a lane a key.
__device__ __forceinline__ void merge_lists(LPShared &s, uint32_t k) {
    const uint32_t lane = threadIdx.x & 31u, warps = blockDim.x / 32;
    for (uint32_t w = threadIdx.x >> 5; w < 2 * LP_MAX_CLUSTER; w += warps) {
        const uint32_t mine = w / 2;
        const uint64_t key = s.sent[mine][lane];
        if (!__any_sync(0xFFFFFFFFu, key != 0)) continue;
        uint32_t before = w % 2 ? 0 : lane;
#pragma unroll
        for (uint32_t x = 0; x < LP_MAX_CLUSTER / 2; ++x) {
            const uint32_t l = w % 2 * (LP_MAX_CLUSTER / 2) + x;
            uint32_t n = 0; // of list l that come before; lists are no longer than 31 or full
#pragma unroll
            for (uint32_t step = 16; step > 0; step >>= 1)
                if (s.sent[l][n + step - 1] > key) n += step;
            n += s.sent[l][n] > key;
            before += l == mine ? 0 : n;
        }
        if (key && before) atomicAdd(&s.before[mine][lane], before);
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < LP_MAX_CLUSTER * 32; i += blockDim.x) {
        const uint64_t key = s.sent[i / 32][i % 32];
        const uint32_t at = s.before[i / 32][i % 32];
        if (key && at < k) s.first[at] = key;
    }
    __syncthreads();
}

// The k first values of the CTA's part of a row, to s.first; `mine` is the key of the thread's
// best chunk, and groups of 2^lanes_log2 threads have put theirs to s.groups.
template <int T>
__device__ __forceinline__ void select_top(const Row<T> &row, const Stream<T> &stream, uint64_t mine, uint64_t group,
                                           uint32_t lanes_log2, uint32_t k, uint32_t rank, uint32_t threads, LPShared &s) {
    constexpr uint32_t V = LP_VEC<T>;
    // the group that k - 1 others come before: its threads share the count
    const uint32_t lanes = 1u << lanes_log2, part = blockDim.x >> (2 * lanes_log2);
    const uint32_t from = (threadIdx.x & (lanes - 1)) * part;
    uint32_t before = 0;
#pragma unroll 8
    for (uint32_t j = 0; j < part; ++j) before += s.groups[from + j] > group;
    for (uint32_t o = 1; o < lanes; o <<= 1) before += __shfl_xor_sync(0xFFFFFFFFu, before, o);
    if (before == k - 1 && group) s.bound = group; // else fewer groups than k have a chunk, and it stays 0
    __syncthreads();
    const uint64_t bound = s.bound;
    const float bound_value = bound ? value_of(static_cast<uint32_t>(bound >> 32)) : -INFINITY;
    const uint32_t bound_chunk = bound ? place_of(bound) : 0xFFFFFFFFu;
    if (mine && mine >= bound) {
        if (stream.second < bound_value)
            s.single[atomicAdd(&s.singles, 1u)] = stream.chunk;
        else
            s.column[atomicAdd(&s.columns, 1u)] = static_cast<uint16_t>(threadIdx.x);
    }
    __syncthreads();
    const uint32_t singles = s.singles, columns = s.columns;
    const uint32_t per = columns ? (row.whole + 2 + threads - 1) / threads : 1, all = singles + columns * per;
    // every value that does not come behind the bound, NaN too
    auto visit = [&](auto &&take) {
        for (uint32_t w = threadIdx.x; w < all; w += blockDim.x) {
            uint32_t chunk;
            if (w < singles) {
                chunk = s.single[w];
            } else {
                const uint32_t c = (w - singles) / per;
                chunk = rank * blockDim.x + s.column[c] + (w - singles - c * per) * threads;
            }
            const uint32_t n = row.size_of(chunk), first = row.first_of(chunk);
            float v[V];
            unpack<T>(chunk - 1 < row.whole ? load_chunk32_again(row.whole_at(chunk - 1)) : row.end(chunk), v);
            const bool ties = chunk <= bound_chunk;
            uint32_t in = 0;
#pragma unroll
            for (uint32_t j = 0; j < V; ++j)
                if (!(ties ? v[j] < bound_value : v[j] <= bound_value)) in |= 1u << j;
            in &= (1u << n) - 1u;
            while (in) {
                const uint32_t j = __ffs(in) - 1;
                in &= in - 1;
                take(key_of(code_of(load1(row.at, T, first + j)), first + j));
            }
        }
    };
    visit([&](uint64_t key) {
        const uint32_t at = atomicAdd(&s.n, 1u);
        if (at < LP_LIST) s.list[at] = key;
    });
    __syncthreads();
    if (s.n <= LP_LIST) {
        rank_keys(s.list, s.n, k, s.first);
    } else {
        // more than the list holds (rows of which a few threads have all the large values): one at a time
        const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
        uint64_t last = ~0ull;
#pragma unroll 1
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
            for (uint32_t w = 0; w < blockDim.x / 32; ++w) last = s.list[w] > last ? s.list[w] : last;
            if (threadIdx.x == 0) s.first[r] = last;
        }
    }
    __syncthreads();
}

// The logarithm of a sum, as that of its exponent and of a value in [3/4, 3/2): f32 for the latter,
// which stays below 0.41, is off by at most 2^-25 (one unit of logf).
__device__ __forceinline__ double log_of(float sum) {
    const int k = static_cast<int>(__float_as_uint(sum) - 0x3F400000u) >> 23; // sum / 2^k in [3/4, 3/2)
    const float near = __uint_as_float(__float_as_uint(sum) - (static_cast<uint32_t>(k) << 23));
    return (sum > 0.0f && sum < INFINITY) ? 0.69314718055994531 * k + static_cast<double>(logf(near))
                                          : static_cast<double>(logf(sum));
}

// FEW: rows that do not fill the GPU, whose threads have two chunks on their way while two are
// added (four of each, and the code that is read once a launch grows: one row of 151936 6.0 us
// without alternatives, 5.2 so).  Where they do, 64 warps an SM are worth more than that (4096
// rows of 128256 in bf16: 192 us with a chunk a thread and 32 registers, 200 with 40, 203 to 211
// with two and 64).
template <int T, bool FEW>
__global__ void __launch_bounds__(FEW ? LP_THREADS : LP_MANY, FEW ? 2 : 8)
    logprobs_kernel(const LogProbParams p, uint32_t ranks) {
    __shared__ LPShared s;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, warps = blockDim.x / 32;
    const uint32_t rank = blockIdx.x % ranks, threads = blockDim.x * ranks;
    const uint64_t r = blockIdx.x / ranks;
    if (threadIdx.x == 0) {
        s.bound = 0;
        s.n = s.singles = s.columns = 0;
    }
    if (threadIdx.x < LP_MAX_TOP) s.first[threadIdx.x] = 0;
    if (ranks > 1) {
        for (uint32_t i = threadIdx.x; i < LP_MAX_CLUSTER * LP_MAX_TOP; i += blockDim.x) {
            s.sent[i / LP_MAX_TOP][i % LP_MAX_TOP] = 0;
            s.before[i / LP_MAX_TOP][i % LP_MAX_TOP] = 0;
        }
        cluster_arrive();
    }
    after_stream();
    let_next();
    const Row<T> row(p, r);
    const uint32_t me = rank * blockDim.x + threadIdx.x;
    const int32_t token = me == 0 ? p.tokens[r] : -1;
    // chunk 0 may be empty, and so may the last
    const uint32_t first = me || row.head ? me : threads, last = row.whole + (row.tail ? 1 : 0);
    Stream<T> stream(p, first <= last ? first : 0xFFFFFFFFu);
    // the warp's lanes have 32 chunks in a row
    const uint32_t total = row.whole + 2;
    uint32_t chunk = me - lane;
    const char *from = row.at + static_cast<int64_t>(row.head * x_size(T)) + (static_cast<int64_t>(me) - 1) * 32;
    auto load = [&](uint32_t first) {
        Chunk x;
        if (first + lane - 1 < row.whole)
            x = load_chunk32(from);
        else
            x = row.end(first + lane);
        from += threads * 32ull;
        return x;
    };
    if constexpr (FEW) {
        // two are added while the next two are on their way
        Chunk x[2], y[2];
        x[0] = load(chunk);
        x[1] = load(chunk + threads);
#pragma unroll 1
        for (; chunk < total; chunk += 2 * threads) {
            y[0] = load(chunk + 2 * threads);
            y[1] = load(chunk + 3 * threads);
            stream.add(p, x[0], chunk + lane);
            stream.add(p, x[1], chunk + threads + lane);
            x[0] = y[0];
            x[1] = y[1];
        }
    } else {
#pragma unroll 1
        for (; chunk < total; chunk += threads) {
            Chunk x = load(chunk);
            stream.add(p, x, chunk + lane);
        }
    }

    // the best chunk, which may be read again, on its way to L1
    if (FEW && p.top && stream.chunk - 1 < row.whole)
        asm volatile("prefetch.global.L1 [%0];\n" ::"l"(row.whole_at(stream.chunk - 1)));
    const bool known = static_cast<uint32_t>(token) < row.vocab; // (of the row's first thread)
    const float given = known ? load1(row.at, T, static_cast<uint32_t>(token)) : 0.0f;
    Sums all = stream.sums();
    // threads a group, and the group's best chunk
    const uint32_t lanes_log2 = blockDim.x > LP_GROUPS ? 31 - __clz(blockDim.x / LP_GROUPS) : 0, lanes = 1u << lanes_log2;
    uint64_t mine = 0, group = 0;
    if (p.top) {
        group = mine = stream.chunk == 0xFFFFFFFFu ? 0 : key_of(code_of(stream.best), stream.chunk);
        for (uint32_t o = 1; o < lanes; o <<= 1) {
            const uint64_t other = __shfl_xor_sync(0xFFFFFFFFu, group, o);
            group = other > group ? other : group;
        }
        if ((threadIdx.x & (lanes - 1)) == 0) s.groups[threadIdx.x >> lanes_log2] = group;
    }
    all.move(warp_max(all.ref), p.c);
    all.sum = warp_sum(all.sum);
    all.tsum = warp_sum(all.tsum);
    if (lane == 0) {
        s.ref[warp] = all.ref;
        s.sum[warp] = all.sum;
        s.tsum[warp] = all.tsum;
    }
    __syncthreads();
    if (p.top) select_top<T>(row, stream, mine, group, lanes_log2, p.top, rank, threads, s);
    if (ranks == 1 && warp) return;
    if (warp == 0) {
        const bool in = lane < warps;
        all.ref = in ? s.ref[lane] : -FLT_MAX;
        all.sum = in ? s.sum[lane] : 0.0f;
        all.tsum = in ? s.tsum[lane] : 0.0f;
        all.move(warp_max(all.ref), p.c);
        all.sum = warp_sum(all.sum);
        all.tsum = warp_sum(all.tsum);
    }
    if (ranks > 1) {
        cluster_wait(); // all CTAs have begun, and the first one has cleared what they send to
        if (threadIdx.x < p.top) cluster_store(smem_u32(&s.sent[rank][threadIdx.x]), 0, s.first[threadIdx.x]);
        if (threadIdx.x == 0) {
            cluster_store(smem_u32(&s.sent_sums[0][rank]), 0, all.ref);
            cluster_store(smem_u32(&s.sent_sums[1][rank]), 0, all.sum);
            cluster_store(smem_u32(&s.sent_sums[2][rank]), 0, all.tsum);
        }
        cluster_arrive();
        cluster_wait();
        if (rank != 0) return;
        if (warp == 0) {
            const bool in = lane < ranks;
            all.ref = in ? s.sent_sums[0][lane] : -FLT_MAX;
            all.sum = in ? s.sent_sums[1][lane] : 0.0f;
            all.tsum = in ? s.sent_sums[2][lane] : 0.0f;
            all.move(warp_max(all.ref), p.c);
            all.sum = warp_sum(all.sum);
            all.tsum = warp_sum(all.tsum);
        }
        if (p.top) merge_lists(s, p.top);
        if (warp) return;
    }
    // sum 0: a row of nothing but -inf
    const double log_sum = log_of(all.sum);
    auto log_p = [&](float x) {
        return all.sum == 0.0f ? -INFINITY : static_cast<float>(p.scale * (static_cast<double>(x) - all.ref) - log_sum);
    };
    if (lane == 0) {
        if (token >= 0 && !known) {
            raise_device_status(p.status, FM_STATUS_INVALID_ARGUMENT);
            p.logprobs[r] = NAN;
        } else {
            p.logprobs[r] = token < 0 ? 0.0f : log_p(given);
        }
        const float h =
            all.sum == 0.0f ? 0.0f : static_cast<float>(log_sum - 0.69314718055994531 * all.tsum / all.sum);
        p.entropy[r] = h < 0.0f ? 0.0f : h;
    }
    if (lane < p.top) {
        const uint64_t key = s.first[lane], at = r * p.top + lane;
        p.top_logprobs[at] = log_p(value_of(static_cast<uint32_t>(key >> 32)));
        p.top_ids[at] = static_cast<int32_t>(place_of(key));
    }
}

template <int T> int launch_logprobs(const LogProbParams &p, const Launch &l, bool few, cudaStream_t s) {
    return launch("logprobs_kernel", few ? logprobs_kernel<T, true> : logprobs_kernel<T, false>, l, s, p, l.cluster);
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
    LogProbParams p{};
    p.logits = a->logits;
    p.stride = a->row_stride;
    p.vocab = a->vocab;
    p.top = a->top;
    p.tokens = a->token;
    p.logprobs = a->logprobs;
    p.entropy = a->entropy;
    p.top_logprobs = a->top_logprobs;
    p.top_ids = a->top_ids;
    p.c = static_cast<float>(a->scale * 1.4426950408889634);
    // 2^t of a raised value is 0 for every reference from `ordinary` on (f16 with small scales
    // has none), and no difference of the short way overflows
    p.raised = a->dtype == FM_X_F16 ? -65504.0f : -std::exp2(std::fmin(std::floor(120.0f - std::log2(p.c)), 100.0f));
    p.ordinary = p.raised * p.c <= 4.0f * LP_LEAST ? p.raised / 2.0f : p.raised - 2.0f * LP_LEAST / p.c;
    p.nothing = -2.0f * LP_LEAST / p.c;
    p.step = 8.0f / p.c;
    p.scale = a->scale;
    p.status = device_status_word();
    // rows that leave SMs idle go to clusters, and to more threads
    const uint64_t chunks = static_cast<uint64_t>(a->vocab) * x_size(a->dtype) / 32;
    const uint64_t sms = static_cast<uint64_t>(device_sm_count());
    uint32_t ranks = 1, threads = 32;
    while (ranks < LP_MAX_CLUSTER && a->tokens * ranks * 2 <= sms && chunks >= ranks * 1024ull) ranks *= 2;
    auto few = [&](uint32_t n) { return static_cast<uint64_t>(a->tokens) * ranks * n <= sms * 1024; };
    while ((threads < LP_MANY && chunks > static_cast<uint64_t>(threads) * ranks * 4) ||
           (threads < LP_THREADS && chunks > static_cast<uint64_t>(threads) * ranks && few(2 * threads)))
        threads *= 2;
    const Launch l{dim3(a->tokens * ranks), threads, 0, ranks, 0};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a->dtype == FM_X_F32) return launch_logprobs<FM_X_F32>(p, l, few(threads), s);
    if (a->dtype == FM_X_BF16) return launch_logprobs<FM_X_BF16>(p, l, few(threads), s);
    return launch_logprobs<FM_X_F16>(p, l, few(threads), s);
}
