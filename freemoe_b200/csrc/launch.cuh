// launch.cuh -- launches that may begin while the kernel before them on the stream still
// runs.  Such a kernel calls after_stream() before it touches memory: it then finds all
// earlier work of the stream done, as it would after an ordinary launch, but its CTAs are
// already there (an ordinary launch costs one to two microseconds between two kernels,
// as much as some of these kernels take).  let_next() lets the next launch of this kind
// come; without it that one begins when this kernel ends.
#pragma once

#include "common.cuh"

namespace fmb {

__device__ __forceinline__ void after_stream() { asm volatile("griddepcontrol.wait;\n" ::: "memory"); }
__device__ __forceinline__ void let_next() { asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory"); }

struct Launch {
    dim3 grid;
    uint32_t threads, smem;
    uint32_t cluster; // CTAs a cluster, 1: none
};
template <typename... K, typename... A>
int launch(const char *what, void (*kernel)(K...), const Launch &l, cudaStream_t s, const A &...args) {
    if (l.smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   static_cast<int>(l.smem));
        if (e != cudaSuccess) return cuda_status(e, what);
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
