// common.cuh — launch helpers shared by the kernel translation units.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

namespace popcorn {
namespace launch {

int current_sm_count();

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

inline int grid_for(int64_t work_items, int threads, int sm_count) {
    int64_t blocks = (work_items + threads - 1) / threads;
    int64_t cap = int64_t(sm_count) * 8;
    if (blocks > cap) blocks = cap;
    return int(blocks < 1 ? 1 : blocks);
}

// Launches with programmatic stream serialisation allowed: the kernel may
// start while its predecessor on the stream drains; every kernel of this
// library calls griddepcontrol.wait before it reads a predecessor's output.
template <class F, class... Args>
cudaError_t launch_k(F kernel, dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// As launch_k, with the grid in clusters of `cluster` CTAs along x.
template <class F, class... Args>
cudaError_t launch_cluster(F kernel, dim3 grid, dim3 block, unsigned cluster, size_t smem, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Runs a kernel's set-up once per device (function attributes belong to the
// device that is current when they are set).
class DeviceOnce {
public:
    template <class F>
    cudaError_t run(F setup) {
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        const uint64_t bit = uint64_t(1) << (dev & 63);
        if (done_.load(std::memory_order_acquire) & bit) return cudaSuccess;
        e = setup();
        if (e == cudaSuccess) done_.fetch_or(bit, std::memory_order_release);
        return e;
    }

private:
    std::atomic<uint64_t> done_{0};
};

// Raises a kernel's dynamic shared memory limit once per process.
template <class F>
cudaError_t allow_smem(F kernel, size_t bytes) {
    if (bytes <= 48 * 1024) return cudaSuccess;
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes));
}

}  // namespace launch
}  // namespace popcorn
