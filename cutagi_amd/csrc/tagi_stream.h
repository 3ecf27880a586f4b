// Loads and stores of W neighbouring floats (one 16-byte access for W = 4), for the kernels
// that pass over their arrays once.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>

namespace tagi {

typedef float stream_floatx4 __attribute__((ext_vector_type(4)));

template <int W>
__device__ __forceinline__ void load_w(const float *p, float (&v)[W]) {
    if (W == 4) {
        const stream_floatx4 q = *reinterpret_cast<const stream_floatx4 *>(p);
#pragma unroll
        for (int c = 0; c < W; c++) v[c] = q[c];
    } else {
        v[0] = p[0];
    }
}
// past_cache: a streaming store
template <int W>
__device__ __forceinline__ void store_w(float *p, const float (&v)[W], bool past_cache) {
    if (W == 4) {
        const stream_floatx4 q = {v[0], v[1 % W], v[2 % W], v[3 % W]};
        if (past_cache)
            __builtin_nontemporal_store(q, reinterpret_cast<stream_floatx4 *>(p));
        else
            *reinterpret_cast<stream_floatx4 *>(p) = q;
    } else {
        p[0] = v[0];
    }
}
// Outputs that the 256 MB memory-side cache cannot hold for whoever reads them next go past
// it, which leaves it to the inputs (layer norm of 16384 x 4096: forward and backward 531 ->
// 517 us, gated sum of 8192 x 4096 with its backward 364 -> 351 us).
inline bool goes_past_cache(size_t output_floats) {
    return output_floats * sizeof(float) >= ((size_t)256 << 20);
}

}  // namespace tagi
