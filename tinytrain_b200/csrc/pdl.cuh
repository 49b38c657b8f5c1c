// Launches that overlap with the end of the kernel before them in the stream
// (programmatic dependent launch): the kernel's blocks may start while that
// kernel drains, and grid_wait() holds them until it has completed and its
// writes are visible. Every kernel launched with launch_pdl() calls
// grid_wait() before it touches global memory.
#pragma once

#include <cuda_runtime.h>

#include "ttk_internal.h"

namespace ttk {

__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <class... P, class... A>
int launch_pdl(const char* what, void (*kernel)(P...), dim3 grid, int threads, size_t smem,
               cudaStream_t st, const A&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
    const int rc = check_launch(what);
    return rc ? rc : check_cuda(e, what);
}

}  // namespace ttk
