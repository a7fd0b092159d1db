// ptx.cuh -- inline-PTX helpers shared by the sm_100a kernels: mbarriers,
// bulk and per-thread async copies, named barriers, clusters.
#pragma once

#include <stdint.h>

namespace fmb {

// ---- mbarriers and bulk copies ------------------------------------------------

__device__ __forceinline__ uint32_t smem_u32(const void *p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ void mbar_init(uint64_t *bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(smem_u32(bar)), "r"(count));
}

__device__ __forceinline__ void mbar_expect_tx(uint64_t *bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(smem_u32(bar)),
                 "r"(bytes)
                 : "memory");
}

__device__ __forceinline__ void mbar_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ bool mbar_try_wait(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}

// Non-blocking test of a phase (no suspension): for a thread that polls several barriers.
__device__ __forceinline__ bool mbar_test_wait(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}

// Bounded wait: false after ~2^31 cycles (about one second) without completion.
__device__ __forceinline__ bool mbar_wait(uint64_t *bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity)) return true;
    const long long start = clock64();
    for (uint32_t it = 1;; ++it) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((it & 255u) == 0 && clock64() - start > (1ll << 31)) return false;
    }
}

__device__ __forceinline__ void bulk_g2s(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(
            smem_u32(dst)),
        "l"(src), "r"(bytes), "r"(smem_u32(bar))
        : "memory");
}

// Arrives on named barrier `id` without waiting (the producer side of a
// bar.arrive / bar.sync pair; `threads` counts both sides).
__device__ __forceinline__ void named_bar_arrive(int id, int threads) {
    asm volatile("bar.arrive %0, %1;\n" ::"r"(id), "r"(threads) : "memory");
}

__device__ __forceinline__ void named_bar_sync(int id, int threads) {
    asm volatile("bar.sync %0, %1;\n" ::"r"(id), "r"(threads) : "memory");
}

// 16-byte per-thread async copy global -> shared (L1 bypassed).
__device__ __forceinline__ void cp_async16(void *dst, const void *src) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;\n" ::"r"(smem_u32(dst)), "l"(src)
                 : "memory");
}

__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }

template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory");
}

// ---- clusters -----------------------------------------------------------------

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_nctarank;\n" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// A value of CTA `rank`'s shared memory, at the address that `addr` has in this one's.
__device__ __forceinline__ float cluster_load(uint32_t addr, uint32_t rank) {
    uint32_t at;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(at) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(v) : "r"(at) : "memory");
    return v;
}

// The two halves of cluster_sync.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory"); }
// Stores to CTA `rank`'s shared memory; all CTAs of the cluster must be known to run.
__device__ __forceinline__ uint32_t cluster_at(uint32_t addr, uint32_t rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(at) : "r"(addr), "r"(rank));
    return at;
}
__device__ __forceinline__ void cluster_store(uint32_t addr, uint32_t rank, uint64_t v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;\n" ::"r"(cluster_at(addr, rank)), "l"(v) : "memory");
}
__device__ __forceinline__ void cluster_store(uint32_t addr, uint32_t rank, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;\n" ::"r"(cluster_at(addr, rank)), "f"(v) : "memory");
}

// ---- arithmetic ---------------------------------------------------------------

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}


// Two f32 values in one register pair, and operations on both.
__device__ __forceinline__ uint64_t pack_f32x2(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpack_f32x2(uint64_t v, float &lo, float &hi) {
    asm("mov.b64 {%0, %1}, %2;\n" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul_f32x2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// Eight values at a time: a *= b, a *= the factor, a = a + b * the factor, sums of squares.
__device__ __forceinline__ void mul8(float (&a)[8], const float (&b)[8]) {
#pragma unroll
    for (int j = 0; j < 8; j += 2)
        unpack_f32x2(mul_f32x2(pack_f32x2(a[j], a[j + 1]), pack_f32x2(b[j], b[j + 1])), a[j], a[j + 1]);
}
__device__ __forceinline__ void mul8(float (&a)[8], float by) {
#pragma unroll
    for (int j = 0; j < 8; j += 2)
        unpack_f32x2(mul_f32x2(pack_f32x2(a[j], a[j + 1]), pack_f32x2(by, by)), a[j], a[j + 1]);
}
__device__ __forceinline__ void add8(float (&a)[8], const float (&b)[8], float by) {
#pragma unroll
    for (int j = 0; j < 8; j += 2)
        unpack_f32x2(fma_f32x2(pack_f32x2(b[j], b[j + 1]), pack_f32x2(by, by), pack_f32x2(a[j], a[j + 1])), a[j], a[j + 1]);
}
__device__ __forceinline__ uint64_t squares8(const float (&a)[8], uint64_t sums) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const uint64_t two = pack_f32x2(a[j], a[j + 1]);
        sums = fma_f32x2(two, two, sums);
    }
    return sums;
}
__device__ __forceinline__ float both(uint64_t sums) {
    float a, b;
    unpack_f32x2(sums, a, b);
    return a + b;
}

} // namespace fmb
