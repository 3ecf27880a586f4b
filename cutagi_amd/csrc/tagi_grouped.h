// Shared by the kernels of the Linear layers grouped by expert.
#pragma once
#include <hip/hip_runtime.h>

namespace tagi {

// Rows [first, end) of expert e, whatever the offsets hold: inside 0..R, never negative.
__device__ __forceinline__ void group_rows(const int *__restrict__ offsets, int e, int R, int &first,
                                           int &end) {
    first = min(max(offsets[e], 0), R);
    end = min(max(offsets[e + 1], first), R);
}

}  // namespace tagi
