// What the paged cache's kernels share.
#pragma once

#include <cuda_runtime.h>

#include "fkv_common.h"

namespace fkvdev {

// A decode step is a chain of small kernels.  Each is launched while its
// predecessor drains (launch_beside) and waits for it before it reads or writes
// anything; after that it lets its own successor start.
__device__ __forceinline__ void await_predecessor() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// a sticky bit of the cache's status word
__device__ __forceinline__ void paged_report(int32_t* status, int bit) {
    if (status != nullptr) atomicOr(status, bit);
}

}  // namespace fkvdev

namespace fkv {

// A launch whose kernel begins with await_predecessor(), early if the grid is
// so small that it finds room beside its predecessor.
template <class... P, class... A>
cudaError_t launch_beside(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t stream, bool early,
                          A... args) {
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = at;
    cfg.numAttrs = early ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Checks a cache descriptor on the host; *pshift = log2(page).
int paged_check(const FkvPagedCache* c, const char* who, int* pshift);

}  // namespace fkv
