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

// Vectors of floats at any float's address: the memory instructions need four bytes only.
typedef float float4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef float float2_any __attribute__((ext_vector_type(2), aligned(4)));

}  // namespace tagi
