// Layer norm of Gaussian activations over the features of each row, gfx950.
//
// Forward, row b:  m = mean_i mu_a,  s = (sum_i (mu_a - m)^2 + sum_i var_a) / (n - 1),
// then the affine map of a normalised Gaussian by Gaussian weights. The statistics are
// taken in two passes over values that stay in registers (the mean first, then squared
// deviations from it), so nothing cancels and HBM is read once.
// Backward: the state innovations are element by element; the parameter innovations are
// sums over the rows, taken in two steps (row chunks, then the chunks in index order: the
// same bits every run, no atomics).
#include <cstdint>

#include "tagi_internal.h"
#include "tagi_stream.h"

namespace tagi {
namespace {

constexpr int TPB = 256;

inline bool aligned16(const void *q) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0; }

// Sums over the THREADS (64 or 256) threads that share a row; every thread gets the result.
template <int THREADS, int NV>
__device__ __forceinline__ void row_sum(float (&v)[NV], float (*s)[TPB / 64]) {
#pragma unroll
    for (int k = 0; k < NV; k++) {
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) v[k] += __shfl_xor(v[k], off, 64);
    }
    if (THREADS == 64) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (lane == 0) {
#pragma unroll
        for (int k = 0; k < NV; k++) s[k][wave] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NV; k++) v[k] = (s[k][0] + s[k][1]) + (s[k][2] + s[k][3]);
    __syncthreads();
}

// ---------------------------------------------------------------------------
// Forward. THREADS threads hold one row, PER groups of W features each (W = 4 where rows
// are whole 16-byte groups, else 1); PER == 0: a row of any length, read three times.
// ---------------------------------------------------------------------------
template <int THREADS, int PER, int W>
__global__ __launch_bounds__(TPB) void ln_fwd_kernel(
    const float *__restrict__ mu_w, const float *__restrict__ var_w,
    const float *__restrict__ mu_b, const float *__restrict__ var_b,
    const float *__restrict__ mu_a, const float *__restrict__ var_a, float epsilon, int n, int B,
    bool past_cache, float *__restrict__ mu_s, float *__restrict__ var_s, float *__restrict__ mu_z,
    float *__restrict__ var_z) {
    __shared__ float s[2][TPB / 64];
    const int t = threadIdx.x % THREADS;
    // (whole waves leave the loop, and whole workgroups where it holds a barrier)
    for (long long b = (long long)blockIdx.x * (TPB / THREADS) + threadIdx.x / THREADS; b < B;
         b += (long long)gridDim.x * (TPB / THREADS)) {
        const float *a = mu_a + (size_t)b * n, *q = var_a + (size_t)b * n;
        const int groups = n / W;
        constexpr int HELD = PER > 0 ? PER : 1;
        float m[HELD][W], v[HELD][W];

        float sum[2] = {0.f, 0.f};
        if (PER > 0) {
#pragma unroll
            for (int i = 0; i < HELD; i++) {
                const int g = i * THREADS + t;
                if (g < groups) {
                    load_w<W>(a + (size_t)g * W, m[i]);
                    load_w<W>(q + (size_t)g * W, v[i]);
                } else {
#pragma unroll
                    for (int c = 0; c < W; c++) m[i][c] = v[i][c] = 0.f;
                }
            }
#pragma unroll
            for (int i = 0; i < HELD; i++)
#pragma unroll
                for (int c = 0; c < W; c++) {
                    sum[0] += m[i][c];
                    sum[1] += v[i][c];
                }
        } else {
            for (int g = t; g < groups; g += THREADS) {
                load_w<W>(a + (size_t)g * W, m[0]);
                load_w<W>(q + (size_t)g * W, v[0]);
#pragma unroll
                for (int c = 0; c < W; c++) {
                    sum[0] += m[0][c];
                    sum[1] += v[0][c];
                }
            }
        }
        row_sum<THREADS, 2>(sum, s);
        const float mean = sum[0] / n;
        float dev[1] = {0.f};
        if (PER > 0) {
#pragma unroll
            for (int i = 0; i < HELD; i++) {
                const bool live = i * THREADS + t < groups;
#pragma unroll
                for (int c = 0; c < W; c++) {
                    const float d = live ? m[i][c] - mean : 0.f;
                    dev[0] += d * d;
                }
            }
        } else {
            for (int g = t; g < groups; g += THREADS) {
                load_w<W>(a + (size_t)g * W, m[0]);
#pragma unroll
                for (int c = 0; c < W; c++) dev[0] += (m[0][c] - mean) * (m[0][c] - mean);
            }
        }
        row_sum<THREADS, 1>(dev, s);
        const float var = (dev[0] + sum[1]) / (n - 1);
        if (t == 0) {
            mu_s[b] = mean;
            var_s[b] = var;
        }
        const float inv = 1.0f / sqrtf(var + epsilon);
        const bool bias = mu_b != nullptr;
        auto one = [&](int g, float (&mi)[W], float (&vi)[W]) {
            const size_t f = (size_t)g * W;
            float mw[W], vw[W], om[W], ov[W];
            load_w<W>(mu_w + f, mw);
            load_w<W>(var_w + f, vw);
#pragma unroll
            for (int c = 0; c < W; c++) {
                const float x = inv * (mi[c] - mean);
                om[c] = x * mw[c];
                ov[c] = inv * inv * vi[c] * (mw[c] * mw[c] + vw[c]) + vw[c] * x * x;
            }
            if (bias) {
                load_w<W>(mu_b + f, mw);
                load_w<W>(var_b + f, vw);
#pragma unroll
                for (int c = 0; c < W; c++) {
                    om[c] += mw[c];
                    ov[c] += vw[c];
                }
            }
            store_w<W>(mu_z + (size_t)b * n + f, om, past_cache);
            store_w<W>(var_z + (size_t)b * n + f, ov, past_cache);
        };
        if (PER > 0) {
#pragma unroll
            for (int i = 0; i < HELD; i++) {
                const int g = i * THREADS + t;
                if (g < groups) one(g, m[i], v[i]);
            }
        } else {
            for (int g = t; g < groups; g += THREADS) {
                load_w<W>(a + (size_t)g * W, m[0]);
                load_w<W>(q + (size_t)g * W, v[0]);
                one(g, m[0], v[0]);
            }
        }
    }
}

// ---------------------------------------------------------------------------
// Backward of one (block of columns, chunk of rows). 2^cw_log threads hold neighbouring
// groups of W columns, the other bits of the thread index are rows. A thread keeps its
// columns' four sums over the rows it walks; the row threads are joined through LDS.
// part: [chunk][4][n].
// ---------------------------------------------------------------------------
template <int W>
__global__ __launch_bounds__(TPB) void ln_bwd_kernel(
    const float *__restrict__ mu_w, const float *__restrict__ mu_a, const float *__restrict__ jcb,
    const float *__restrict__ mu_s, const float *__restrict__ var_s,
    const float *__restrict__ dmu_out, const float *__restrict__ dvar_out, float epsilon, int n,
    int B, int rows_per_chunk, int cw_log, int state_update, int param_update, bool past_cache,
    float *__restrict__ dmu, float *__restrict__ dvar, float *__restrict__ part) {
    __shared__ float s[4][W][TPB];
    const int cw = 1 << cw_log;
    const int ct = threadIdx.x & (cw - 1), rt = threadIdx.x >> cw_log, row_step = TPB >> cw_log;
    const int g = blockIdx.x * cw + ct;
    const bool live = g < n / W;
    const size_t f = (size_t)(live ? g : 0) * W;
    const int b_lo = blockIdx.y * rows_per_chunk, b_hi = min(B, b_lo + rows_per_chunk);
    float mw[W], acc[4][W];
    load_w<W>(mu_w + f, mw);
#pragma unroll
    for (int k = 0; k < 4; k++)
#pragma unroll
        for (int c = 0; c < W; c++) acc[k][c] = 0.f;
    if (live) {
        for (int b = b_lo + rt; b < b_hi; b += row_step) {
            const size_t at = (size_t)b * n + f;
            float dm[W], dv[W];
            load_w<W>(dmu_out + at, dm);
            load_w<W>(dvar_out + at, dv);
            const float inv = 1.0f / sqrtf(var_s[b] + epsilon);
            if (state_update) {
                float t[W], om[W], ov[W];
                if (jcb != nullptr) {
                    load_w<W>(jcb + at, t);
                } else {
#pragma unroll
                    for (int c = 0; c < W; c++) t[c] = 1.f;
                }
#pragma unroll
                for (int c = 0; c < W; c++) {
                    t[c] *= inv * mw[c];
                    om[c] = t[c] * dm[c];
                    ov[c] = t[c] * dv[c] * t[c];
                }
                store_w<W>(dmu + at, om, past_cache);
                store_w<W>(dvar + at, ov, past_cache);
            }
            if (param_update) {
                float x[W];
                load_w<W>(mu_a + at, x);
                const float mean = mu_s[b];
#pragma unroll
                for (int c = 0; c < W; c++) {
                    x[c] = inv * (x[c] - mean);
                    acc[0][c] += x[c] * dm[c];
                    acc[1][c] += x[c] * x[c] * dv[c];
                    acc[2][c] += dm[c];
                    acc[3][c] += dv[c];
                }
            }
        }
    }
    if (!param_update) return;
#pragma unroll
    for (int k = 0; k < 4; k++)
#pragma unroll
        for (int c = 0; c < W; c++) s[k][c][threadIdx.x] = acc[k][c];
    __syncthreads();
    if (rt == 0 && live) {
        float *o = part + (size_t)blockIdx.y * 4 * n + f;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            float v[W];
#pragma unroll
            for (int c = 0; c < W; c++) {
                v[c] = 0.f;
                for (int r = 0; r < row_step; r++) v[c] += s[k][c][(r << cw_log) + ct];
            }
#pragma unroll
            for (int c = 0; c < W; c++) o[(size_t)k * n + c] = v[c];
        }
    }
}

// The chunks of 64 columns: sixteen waves take every sixteenth chunk, their sums are joined in
// wave order.
constexpr int FINAL_WAVES = 16;
__global__ __launch_bounds__(FINAL_WAVES * 64) void ln_bwd_final_kernel(
    const float *__restrict__ part, const float *__restrict__ var_w,
    const float *__restrict__ var_b, int n, int chunks, float *__restrict__ dmu_w,
    float *__restrict__ dvar_w, float *__restrict__ dmu_b, float *__restrict__ dvar_b) {
    __shared__ float s[4][FINAL_WAVES][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int c = blockIdx.x * 64 + lane;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < n)
        for (int q = wave; q < chunks; q += FINAL_WAVES) {
            const float *o = part + (size_t)q * 4 * n + c;
#pragma unroll
            for (int k = 0; k < 4; k++) v[k] += o[(size_t)k * n];
        }
#pragma unroll
    for (int k = 0; k < 4; k++) s[k][wave][lane] = v[k];
    __syncthreads();
    if (wave != 0 || c >= n) return;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        v[k] = 0.f;
#pragma unroll
        for (int w = 0; w < FINAL_WAVES; w++) v[k] += s[k][w][lane];
    }
    const float vw = var_w[c];
    dmu_w[c] = vw * v[0];
    dvar_w[c] = vw * vw * v[1];
    if (var_b != nullptr) {
        const float vb = var_b[c];
        dmu_b[c] = vb * v[2];
        dvar_b[c] = vb * vb * v[3];
    }
}

// Launch shape of the backward pass: columns per workgroup and rows per chunk, from n and B
// alone, so that the scratch size does not depend on the pointers. `groups` is n / 4 where n
// is a multiple of four; unaligned arrays then take the one-column form with the same chunks.
int ln_rows_per_chunk(int n, int B) {
    const long long col_blocks = (n + 255) / 256;
    // four workgroups per CU (16384 x 4096, forward and backward: 2 / 3 / 4 / 8 / 16 per CU take
    // 540 / 497 / 493 / 517 / 508 us; more of them also leave more partial sums)
    long long chunks = (4LL * num_cu() + col_blocks - 1) / col_blocks;
    long long rows = (B + chunks - 1) / chunks;
    if (rows < 16) rows = 16;
    return (int)rows;
}

template <int THREADS, int PER, int W>
hipError_t fwd(const float *mu_w, const float *var_w, const float *mu_b, const float *var_b,
               const float *mu_a, const float *var_a, float epsilon, int n, int B, float *mu_s,
               float *var_s, float *mu_z, float *var_z, hipStream_t stream) {
    // (a launch holds fewer than 2^32 threads; beyond that the workgroups walk on)
    const long long rows = TPB / THREADS, blocks = (B + rows - 1) / rows;
    const unsigned grid = (unsigned)(blocks < (1 << 22) ? blocks : 1 << 22);
    hipLaunchKernelGGL((ln_fwd_kernel<THREADS, PER, W>), dim3(grid), dim3(TPB), 0, stream, mu_w, var_w, mu_b, var_b, mu_a, var_a, epsilon, n, B,
                       goes_past_cache((size_t)2 * B * n), mu_s, var_s, mu_z, var_z);
    return hipGetLastError();
}

}  // namespace

size_t layernorm_bwd_scratch_floats(int n, int B) {
    const int rows = ln_rows_per_chunk(n, B);
    return (size_t)((B + rows - 1) / rows) * 4 * n;
}

hipError_t launch_layernorm_fwd(const float *mu_w, const float *var_w, const float *mu_b,
                                const float *var_b, const float *mu_a, const float *var_a,
                                float epsilon, int n, int B, float *mu_s, float *var_s,
                                float *mu_z, float *var_z, hipStream_t stream) {
    const bool vec = n % 4 == 0 && aligned16(mu_w) && aligned16(var_w) && aligned16(mu_b) &&
                     aligned16(var_b) && aligned16(mu_a) && aligned16(var_a) && aligned16(mu_z) &&
                     aligned16(var_z);
#define LN_FWD(T, P, W)                                                                          \
    return fwd<T, P, W>(mu_w, var_w, mu_b, var_b, mu_a, var_a, epsilon, n, B, mu_s, var_s, mu_z, \
                        var_z, stream)
    // One wave per row up to 1024 features, unless the rows would not fill the chip that way
    // (four waves for every SIMD): then a workgroup each.
    const bool many = B >= 16 * num_cu();
    if (vec) {
        if (n <= 256) LN_FWD(64, 1, 4);
        if (n <= 1024 && many) LN_FWD(64, 4, 4);
        if (n <= 1024) LN_FWD(256, 1, 4);
        if (n <= 4096) LN_FWD(256, 4, 4);
        if (n <= 8192) LN_FWD(256, 8, 4);
        LN_FWD(256, 0, 4);
    }
    if (n <= 256) LN_FWD(64, 4, 1);
    if (n <= 1024 && many) LN_FWD(64, 16, 1);
    if (n <= 1024) LN_FWD(256, 4, 1);
    if (n <= 4096) LN_FWD(256, 16, 1);
    if (n <= 8192) LN_FWD(256, 32, 1);
    LN_FWD(256, 0, 1);
#undef LN_FWD
}

hipError_t launch_layernorm_bwd(const float *mu_w, const float *var_w, const float *var_b,
                                const float *mu_a, const float *jcb, const float *mu_s,
                                const float *var_s, const float *dmu_out, const float *dvar_out,
                                float epsilon, int n, int B, int state_update, int param_update,
                                float *scratch, float *dmu, float *dvar, float *dmu_w,
                                float *dvar_w, float *dmu_b, float *dvar_b, hipStream_t stream) {
    const bool vec = n % 4 == 0 && aligned16(mu_w) && aligned16(dmu_out) && aligned16(dvar_out) &&
                     (!state_update || (aligned16(jcb) && aligned16(dmu) && aligned16(dvar))) &&
                     (!param_update || aligned16(mu_a));
    const bool past_cache = goes_past_cache((size_t)2 * B * n);
    const int rows = ln_rows_per_chunk(n, B);
    const int chunks = (B + rows - 1) / rows, groups = vec ? n / 4 : n;
    int cw_log = 0;
    while (cw_log < 6 && (1 << cw_log) < groups) cw_log++;
    const dim3 grid((groups + (1 << cw_log) - 1) >> cw_log, chunks);
    if (vec)
        hipLaunchKernelGGL(ln_bwd_kernel<4>, grid, dim3(TPB), 0, stream, mu_w, mu_a, jcb, mu_s,
                           var_s, dmu_out, dvar_out, epsilon, n, B, rows, cw_log, state_update,
                           param_update, past_cache, dmu, dvar, scratch);
    else
        hipLaunchKernelGGL(ln_bwd_kernel<1>, grid, dim3(TPB), 0, stream, mu_w, mu_a, jcb, mu_s,
                           var_s, dmu_out, dvar_out, epsilon, n, B, rows, cw_log, state_update,
                           param_update, past_cache, dmu, dvar, scratch);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !param_update) return e;
    hipLaunchKernelGGL(ln_bwd_final_kernel, dim3((n + 63) / 64), dim3(FINAL_WAVES * 64), 0, stream,
                       scratch,
                       var_w, var_b, n, chunks, dmu_w, dvar_w, dmu_b, dvar_b);
    return hipGetLastError();
}

}  // namespace tagi
