// Launches whose kernels may begin while the one before them on the stream ends, and what such kernels share.
#pragma once
#include "common.cuh"

namespace znn {

// Returns when the kernel before this one on the stream has ended and what it wrote can be read: called before a kernel reads or writes
// anything.  The launch itself then costs no time between the two (norm and Adam step of 2 million floats: 15.0 us a call, 18.7 without).
__device__ __forceinline__ void wait_for_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// sum over a block of up to 1024 threads in a fixed order, valid in every thread; sh: a double per warp
__device__ __forceinline__ double block_sum(double v, double* sh)
{
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (lane == 0) sh[w] = v;
    __syncthreads();
    double t = 0.0;
    for (int i = 0; i < nw; i++) t += sh[i];
    return t;
}

// Launches `kernel`, which calls wait_for_previous_kernel(), in clusters of `ranks` blocks (1: as its attributes say).
template <class... Params, class... Args>
int launch_overlapped(void (*kernel)(Params...), const char* name, size_t blocks, int threads, int ranks, const Args&... args)
{
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(threads);
    cfg.stream = stream();
    cudaLaunchAttribute attrs[2] = {};
    if (ranks > 1) {
        attrs[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attrs[cfg.numAttrs++].val.clusterDim = {(unsigned)ranks, 1, 1};
    }
    attrs[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attrs;
    ZNN_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, args...));
    ZNN_LAUNCH_OK(name);
    return ZNN_OK;
}

}  // namespace znn
