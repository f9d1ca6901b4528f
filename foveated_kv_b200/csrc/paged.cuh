// What the paged cache's kernels share.
#pragma once

#include <cuda_runtime.h>

#include "fkv_common.h"

namespace fkvdev {

// a sticky bit of the cache's status word
__device__ __forceinline__ void paged_report(int32_t* status, int bit) {
    if (status != nullptr) atomicOr(status, bit);
}

}  // namespace fkvdev

namespace fkv {

// Checks a cache descriptor on the host; *pshift = log2(page).
int paged_check(const FkvPagedCache* c, const char* who, int* pshift);

}  // namespace fkv
