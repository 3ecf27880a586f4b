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

// The slot-th group of up to `rows` rows over all experts, for a wave: expert (-1 behind the
// last), first row, end of the expert's rows. There are at most R / rows + min(E, R) of them.
__device__ __forceinline__ int find_rows(const int *__restrict__ offsets, int E, int R, int rows,
                                         int slot, int &r0, int &end) {
    const int lane = threadIdx.x & 63;
    int carry = 0;
    for (int e0 = 0; e0 < E; e0 += 64) {
        int first = 0, last = 0;
        if (e0 + lane < E) group_rows(offsets, e0 + lane, R, first, last);
        const int groups = (last - first + rows - 1) / rows;
        int inc = groups;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int u = __shfl_up(inc, off, 64);
            if (lane >= off) inc += u;
        }
        const unsigned long long reach = __ballot(carry + inc > slot);
        if (reach != 0ull) {
            const int at = __ffsll(reach) - 1;
            const int before = carry + __builtin_amdgcn_readlane(inc - groups, at);
            r0 = __builtin_amdgcn_readlane(first, at) + (slot - before) * rows;
            end = __builtin_amdgcn_readlane(last, at);
            return e0 + at;
        }
        carry += __builtin_amdgcn_readlane(inc, 63);
    }
    return -1;
}

// Vectors of floats at any float's address: the memory instructions need four bytes only.
typedef float float4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef float float2_any __attribute__((ext_vector_type(2), aligned(4)));

}  // namespace tagi
