// launch.cuh -- launches that may begin while the kernel before them on the stream still
// runs.  Such a kernel calls after_stream() before it touches memory: it then finds all
// earlier work of the stream done, as it would after an ordinary launch, but its CTAs are
// already there (an ordinary launch costs one to two microseconds between two kernels,
// as much as some of these kernels take).  let_next() lets the next launch of this kind
// come; without it that one begins when this kernel ends.  Such kernels read memory by ordinary
// loads: read-only ones (ld.global.nc, __ldg) promise data that nobody writes from the kernel's
// begin on, which is before after_stream(), and may be moved there.
#pragma once

#include "common.cuh"

namespace fmb {

__device__ __forceinline__ void after_stream() { asm volatile("griddepcontrol.wait;\n" ::: "memory"); }
__device__ __forceinline__ void let_next() { asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory"); }

struct Launch {
    dim3 grid;
    uint32_t threads, smem;
    uint32_t cluster; // CTAs a cluster, 1: none
    uint32_t most;    // the most shared memory that any launch of this kernel asks for
};
// A launch may have 48 KB without asking, a kernel's static share among them: from here on the limit
// of the dynamic share is raised.
constexpr uint32_t ASK_FOR_SMEM = 32 * 1024;

// The limit belongs to the kernel and not to the launch, and other host threads may be between
// theirs and their launches: every launch that needs one sets the same, the most that any needs.
template <typename... K> cudaError_t allow_smem(void (*kernel)(K...), const Launch &l) {
    if (l.smem <= ASK_FOR_SMEM) return cudaSuccess;
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(l.most));
}

// CTAs of such launches that an SM holds.
template <typename... K> uint32_t ctas_per_sm(void (*kernel)(K...), const Launch &l) {
    int n = 0;
    if (allow_smem(kernel, l) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, static_cast<int>(l.threads), l.smem) != cudaSuccess || n < 1) {
        (void)cudaGetLastError();
        n = 1;
    }
    return static_cast<uint32_t>(n);
}

template <typename... K, typename... A>
int launch(const char *what, void (*kernel)(K...), const Launch &l, cudaStream_t s, const A &...args) {
    const cudaError_t limit = allow_smem(kernel, l);
    if (limit != cudaSuccess) {
        (void)cudaGetLastError();
        return cuda_status(limit, what);
    }
    cudaLaunchAttribute attrs[2]{};
    cudaLaunchConfig_t config{};
    config.gridDim = l.grid;
    config.blockDim = dim3(l.threads);
    config.dynamicSmemBytes = l.smem;
    config.stream = s;
    config.attrs = attrs;
    attrs[config.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[config.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    if (l.cluster > 1) {
        attrs[config.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attrs[config.numAttrs].val.clusterDim.x = l.cluster;
        attrs[config.numAttrs].val.clusterDim.y = attrs[config.numAttrs].val.clusterDim.z = 1;
        ++config.numAttrs;
    }
    const cudaError_t err = cudaLaunchKernelEx(&config, kernel, args...);
    if (err != cudaSuccess) {
        (void)cudaGetLastError();
        return cuda_status(err, what);
    }
    return FM_STATUS_OK;
}

} // namespace fmb
