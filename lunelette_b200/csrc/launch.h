// Kernel launches with programmatic dependent launch (PDL): a kernel may start
// while the previous kernel of the stream finishes; it runs griddepcontrol.wait
// (pdl_wait) before touching anything that kernel wrote. LUNELETTE_PDL=0 turns
// the attribute off for comparisons.
#pragma once
#include <atomic>
#include <cuda_runtime.h>
#include <stdlib.h>

namespace lun {

inline bool pdl_enabled()
{
    static const bool on = [] {
        const char *v = getenv("LUNELETTE_PDL");
        return !(v && v[0] == '0');
    }();
    return on;
}

template <typename... Params, typename... Args>
cudaError_t launch(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                   Args &&...args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<Args &&>(args)...);
}

// The same in clusters of `ranks` blocks (the grid a multiple of it).
template <typename... Params, typename... Args>
cudaError_t launch_cluster(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, int ranks, cudaStream_t stream,
                           Args &&...args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<Args &&>(args)...);
}

// Dynamic shared memory above 48 KB (and clusters of more than 8 blocks) for a kernel,
// set once per kernel and device; safe from several threads.
template <auto Kernel> cudaError_t opt_in(int smem, bool large_clusters = false)
{
    static std::atomic<unsigned long long> done[2];  // devices 0..127
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const bool known = dev >= 0 && dev < 128;
    const unsigned long long bit = 1ull << (dev & 63);
    if (known && (done[dev >> 6].load(std::memory_order_acquire) & bit)) return cudaSuccess;
    e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess && large_clusters)
        e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess && known) done[dev >> 6].fetch_or(bit, std::memory_order_release);
    return e;
}

}  // namespace lun
