// Loads and stores of four neighbouring floats at any float's address, for the kernels that
// pass over the rows of their arrays once: a row of any length is groups of four and one part
// group.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>

namespace tagi {

// (the memory instructions need four bytes only)
typedef float stream4 __attribute__((ext_vector_type(4), aligned(4)));

// Elements 4 g .. 4 g + 3 that a row of n has: 0 to 4.
__device__ __forceinline__ int in_group(int g, int n) { return min(max(n - 4 * g, 0), 4); }

// `valid` floats from p on, zeros behind them
__device__ __forceinline__ void load_group(const float *p, int valid, float (&v)[4]) {
    if (valid == 4) {
        const stream4 q = *reinterpret_cast<const stream4 *>(p);
#pragma unroll
        for (int c = 0; c < 4; c++) v[c] = q[c];
    } else {
#pragma unroll
        for (int c = 0; c < 4; c++) v[c] = c < valid ? p[c] : 0.f;
    }
}
// past_cache: a streaming store
__device__ __forceinline__ void store_group(float *p, int valid, const float (&v)[4], bool past_cache) {
    if (valid == 4) {
        const stream4 q = {v[0], v[1], v[2], v[3]};
        if (past_cache)
            __builtin_nontemporal_store(q, reinterpret_cast<stream4 *>(p));
        else
            *reinterpret_cast<stream4 *>(p) = q;
    } else {
#pragma unroll
        for (int c = 0; c < 3; c++)
            if (c < valid) p[c] = v[c];
    }
}
// Outputs that the 256 MB memory-side cache cannot hold for whoever reads them next go past
// it, which leaves it to the inputs (layer norm of 16384 x 4096: forward and backward 531 ->
// 517 us, gated sum of 8192 x 4096 with its backward 364 -> 351 us).
inline bool goes_past_cache(size_t output_floats) {
    return output_floats * sizeof(float) >= ((size_t)256 << 20);
}

}  // namespace tagi
