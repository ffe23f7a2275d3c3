// Host side of the decode operators: the GPU of a context made current for the duration of a call, and launches that may be set up
// while the kernel before them still runs.
#pragma once
#include <cuda_runtime.h>

#include "context.h"

// Makes a context's GPU current and puts the caller's current device back afterwards.

struct S1DeviceGuard {
    int before = -1;
    bool ok = false;
    explicit S1DeviceGuard(int device) {
        ok = cudaGetDevice(&before) == cudaSuccess;
        if (ok && before != device) ok = cudaSetDevice(device) == cudaSuccess;
        else before = -1;
    }
    ~S1DeviceGuard() {
        if (before >= 0) cudaSetDevice(before);
    }
    S1DeviceGuard(const S1DeviceGuard&) = delete;
    S1DeviceGuard& operator=(const S1DeviceGuard&) = delete;
};

// Launches a kernel that waits (griddepcontrol.wait) before it touches memory, with programmatic stream serialization unless the
// context's "pdl" option is off: a step of a decoder is a chain of kernels of a few microseconds, and their set-up then lies under
// the kernel before. Such a kernel reads what others may have written with plain loads: its blocks can be there while the kernel
// before still reads and writes on the same SM, and the read-only path promises nothing about data that changes in a kernel's life.
template <typename Params>
inline cudaError_t s1_launch_waiting(s1_ctx* ctx, void (*kernel)(Params), unsigned grid_x, unsigned grid_y, unsigned threads, size_t smem,
                                     const Params& params, unsigned cluster = 1) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    unsigned n = 0;
    if (ctx->opt_pdl) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = cluster, attr[n].val.clusterDim.y = 1, attr[n++].val.clusterDim.z = 1;
    }
    cfg.gridDim = dim3(grid_x, grid_y), cfg.blockDim = dim3(threads), cfg.dynamicSmemBytes = smem, cfg.stream = ctx->stream;
    cfg.attrs = attr, cfg.numAttrs = n;
    return cudaLaunchKernelEx(&cfg, kernel, params);
}
