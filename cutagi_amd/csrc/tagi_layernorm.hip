// Layer norm of Gaussian activations over the features of each row, gfx950.
//
// Forward, row b:  m = mean_i mu_a,  s = (sum_i (mu_a - m)^2 + sum_i var_a) / (n - 1),
// then the affine map of a normalised Gaussian by Gaussian weights. The statistics are
// taken in two passes over values that stay in registers (the mean first, then squared
// deviations from it), so nothing cancels and HBM is read once.
// Backward: the state innovations are element by element; the parameter innovations are
// sums over the rows, taken in two steps (row chunks, then the chunks in index order: the
// same bits every run, no atomics).
#include "tagi_internal.h"
#include "tagi_stream.h"

namespace tagi {
namespace {

constexpr int TPB = 256;

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
// Forward. THREADS threads hold one row, PER groups of four features each; PER == 0: a row of
// any length, read three times. Bound by memory, 16 bytes per element: 16384 x 4096 in 195 us,
// 5.5 TB/s.
// ---------------------------------------------------------------------------
template <int THREADS, int PER>
__global__ __launch_bounds__(TPB) void ln_fwd_kernel(
    const float *__restrict__ mu_w, const float *__restrict__ var_w,
    const float *__restrict__ mu_b, const float *__restrict__ var_b,
    const float *__restrict__ mu_a, const float *__restrict__ var_a, float epsilon, int n, int B,
    bool past_cache, float *__restrict__ mu_s, float *__restrict__ var_s, float *__restrict__ mu_z,
    float *__restrict__ var_z) {
    __shared__ float s[2][TPB / 64];
    const int t = threadIdx.x % THREADS;
    const int groups = (n + 3) / 4;
    constexpr int HELD = PER > 0 ? PER : 1;
    // (whole waves leave the loop, and whole workgroups where it holds a barrier)
    for (long long b = (long long)blockIdx.x * (TPB / THREADS) + threadIdx.x / THREADS; b < B;
         b += (long long)gridDim.x * (TPB / THREADS)) {
        const float *a = mu_a + (size_t)b * n, *q = var_a + (size_t)b * n;
        float m[HELD][4], v[HELD][4];

        float sum[2] = {0.f, 0.f};
        auto add = [&](const float (&mi)[4], const float (&vi)[4]) {
            sum[0] += (mi[0] + mi[1]) + (mi[2] + mi[3]);
            sum[1] += (vi[0] + vi[1]) + (vi[2] + vi[3]);
        };
        if (PER > 0) {
#pragma unroll
            for (int i = 0; i < HELD; i++) {
                const int g = i * THREADS + t, valid = in_group(g, n);
                load_group(a + (size_t)g * 4, valid, m[i]);
                load_group(q + (size_t)g * 4, valid, v[i]);
            }
#pragma unroll
            for (int i = 0; i < HELD; i++) add(m[i], v[i]);
        } else {
            for (int g = t; g < groups; g += THREADS) {
                load_group(a + (size_t)g * 4, in_group(g, n), m[0]);
                load_group(q + (size_t)g * 4, in_group(g, n), v[0]);
                add(m[0], v[0]);
            }
        }
        row_sum<THREADS, 2>(sum, s);
        const float mean = sum[0] / n;
        float dev[1] = {0.f};
        auto deviate = [&](const float (&mi)[4], int valid) {
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const float d = c < valid ? mi[c] - mean : 0.f;
                dev[0] += d * d;
            }
        };
        if (PER > 0) {
#pragma unroll
            for (int i = 0; i < HELD; i++) deviate(m[i], in_group(i * THREADS + t, n));
        } else {
            for (int g = t; g < groups; g += THREADS) {
                load_group(a + (size_t)g * 4, in_group(g, n), m[0]);
                deviate(m[0], in_group(g, n));
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
        auto one = [&](int g, const float (&mi)[4], const float (&vi)[4]) {
            const size_t f = (size_t)g * 4;
            const int valid = in_group(g, n);
            float mw[4], vw[4], om[4], ov[4];
            load_group(mu_w + f, valid, mw);
            load_group(var_w + f, valid, vw);
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const float x = inv * (mi[c] - mean);
                om[c] = x * mw[c];
                ov[c] = inv * inv * vi[c] * (mw[c] * mw[c] + vw[c]) + vw[c] * x * x;
            }
            if (bias) {
                load_group(mu_b + f, valid, mw);
                load_group(var_b + f, valid, vw);
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    om[c] += mw[c];
                    ov[c] += vw[c];
                }
            }
            store_group(mu_z + (size_t)b * n + f, valid, om, past_cache);
            store_group(var_z + (size_t)b * n + f, valid, ov, past_cache);
        };
        if (PER > 0) {
#pragma unroll
            for (int i = 0; i < HELD; i++) {
                const int g = i * THREADS + t;
                if (g < groups) one(g, m[i], v[i]);
            }
        } else {
            for (int g = t; g < groups; g += THREADS) {
                load_group(a + (size_t)g * 4, in_group(g, n), m[0]);
                load_group(q + (size_t)g * 4, in_group(g, n), v[0]);
                one(g, m[0], v[0]);
            }
        }
    }
}

// ---------------------------------------------------------------------------
// Backward of one (block of columns, chunk of rows). 2^cw_log threads (up to a wave) hold
// neighbouring groups of four columns, the other bits of the thread index are rows. A thread
// keeps its columns' four sums over the rows it walks; the row threads of a wave are joined by
// lane exchanges, the waves through LDS. The sums go to part ([chunk][4][n]), or where there is
// one chunk only to the innovations. Bound by memory, 24 bytes per element: 16384 x 4096 in 310
// us, 5.2 TB/s.
// ---------------------------------------------------------------------------
struct ParamOut {
    const float *var_w, *var_b;
    float *dmu_w, *dvar_w, *dmu_b, *dvar_b;
};
__global__ __launch_bounds__(TPB) void ln_bwd_kernel(
    const float *__restrict__ mu_w, const float *__restrict__ mu_a, const float *__restrict__ jcb,
    const float *__restrict__ mu_s, const float *__restrict__ var_s,
    const float *__restrict__ dmu_out, const float *__restrict__ dvar_out, float epsilon, int n,
    int B, int rows_per_chunk, int cw_log, int state_update, int param_update, bool past_cache,
    float *__restrict__ dmu, float *__restrict__ dvar, float *__restrict__ part, ParamOut out) {
    __shared__ float s[TPB / 64][16][64];
    const int cw = 1 << cw_log, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int ct = threadIdx.x & (cw - 1), rt = threadIdx.x >> cw_log, row_step = TPB >> cw_log;
    const int g = blockIdx.x * cw + ct, valid = in_group(g, n);
    const size_t f = (size_t)g * 4;
    const int b_lo = blockIdx.y * rows_per_chunk, b_hi = min(B, b_lo + rows_per_chunk);
    float mw[4], acc[4][4];
    load_group(mu_w + f, valid, mw);
#pragma unroll
    for (int k = 0; k < 4; k++)
#pragma unroll
        for (int c = 0; c < 4; c++) acc[k][c] = 0.f;
    if (valid > 0) {
        for (int b = b_lo + rt; b < b_hi; b += row_step) {
            const size_t at = (size_t)b * n + f;
            float dm[4], dv[4];
            load_group(dmu_out + at, valid, dm);
            load_group(dvar_out + at, valid, dv);
            const float inv = 1.0f / sqrtf(var_s[b] + epsilon);
            if (state_update) {
                float t[4], om[4], ov[4];
                if (jcb != nullptr) {
                    load_group(jcb + at, valid, t);
                } else {
#pragma unroll
                    for (int c = 0; c < 4; c++) t[c] = 1.f;
                }
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    t[c] *= inv * mw[c];
                    om[c] = t[c] * dm[c];
                    ov[c] = t[c] * dv[c] * t[c];
                }
                store_group(dmu + at, valid, om, past_cache);
                store_group(dvar + at, valid, ov, past_cache);
            }
            if (param_update) {
                float x[4];
                load_group(mu_a + at, valid, x);
                const float mean = mu_s[b];
#pragma unroll
                for (int c = 0; c < 4; c++) {
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
    for (int off = 32; off >= cw; off >>= 1)
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int c = 0; c < 4; c++) acc[k][c] += __shfl_xor(acc[k][c], off, 64);
    if (lane < cw)
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int c = 0; c < 4; c++) s[wave][4 * k + c][lane] = acc[k][c];
    __syncthreads();
    // thread: sum k of column group ct (256 threads: four sums of 64 groups)
    for (int i = threadIdx.x; i < 4 * cw; i += TPB) {
        const int k = i >> cw_log, at = i & (cw - 1), have = in_group(blockIdx.x * cw + at, n);
        float v[4];
#pragma unroll
        for (int c = 0; c < 4; c++)
            v[c] = (s[0][4 * k + c][at] + s[1][4 * k + c][at]) + (s[2][4 * k + c][at] + s[3][4 * k + c][at]);
        const size_t col = (size_t)(blockIdx.x * cw + at) * 4;
        if (gridDim.y > 1) {
            store_group(part + ((size_t)blockIdx.y * 4 + k) * n + col, have, v, false);
            continue;
        }
        if (k >= 2 && out.var_b == nullptr) continue;
        float f[4];
        load_group((k < 2 ? out.var_w : out.var_b) + col, have, f);
#pragma unroll
        for (int c = 0; c < 4; c++) v[c] *= k & 1 ? f[c] * f[c] : f[c];
        store_group((k == 0 ? out.dmu_w : k == 1 ? out.dvar_w : k == 2 ? out.dmu_b : out.dvar_b) + col, have, v, false);
    }
}

// The chunks of 2^cw_log (up to 64) columns: the other bits of the thread index share out the
// chunks; their sums are joined like the row threads' above.
constexpr int FINAL_WAVES = 16;
__global__ __launch_bounds__(FINAL_WAVES * 64) void ln_bwd_final_kernel(const float *__restrict__ part, int n,
                                                                       int chunks, int cw_log, ParamOut out) {
    __shared__ float s[4][FINAL_WAVES][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, cw = 1 << cw_log;
    const int c = blockIdx.x * cw + (threadIdx.x & (cw - 1));
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < n)
        for (int q = threadIdx.x >> cw_log; q < chunks; q += (FINAL_WAVES * 64) >> cw_log) {
            const float *o = part + (size_t)q * 4 * n + c;
#pragma unroll
            for (int k = 0; k < 4; k++) v[k] += o[(size_t)k * n];
        }
    for (int off = 32; off >= cw; off >>= 1)
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] += __shfl_xor(v[k], off, 64);
#pragma unroll
    for (int k = 0; k < 4; k++) s[k][wave][lane] = v[k];
    __syncthreads();
    if (threadIdx.x >= cw || c >= n) return;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        v[k] = 0.f;
#pragma unroll
        for (int w = 0; w < FINAL_WAVES; w++) v[k] += s[k][w][lane];
    }
    const float vw = out.var_w[c];
    out.dmu_w[c] = vw * v[0];
    out.dvar_w[c] = vw * vw * v[1];
    if (out.var_b != nullptr) {
        const float vb = out.var_b[c];
        out.dmu_b[c] = vb * v[2];
        out.dvar_b[c] = vb * vb * v[3];
    }
}

// Threads that hold neighbouring groups of columns, and rows per chunk: from n and B alone.
int ln_cw_log(int n) {
    int l = 0;
    while (l < 6 && (1 << l) < (n + 3) / 4) l++;
    return l;
}
struct LnChunks {
    int rows, most;   // rows of a chunk, chunks at most (never more for fewer rows)
};
LnChunks ln_chunks(int n, int B) {
    // four workgroups per CU (16384 x 4096, forward and backward: 2 / 3 / 4 / 8 / 16 per CU take
    // 540 / 497 / 493 / 517 / 508 us; more of them also leave more partial sums), but four rows
    // for every row thread (sixteen in all at least)
    const int cw = 1 << ln_cw_log(n);
    const long long col_blocks = ((n + 3) / 4 + cw - 1) / cw;
    const long long chunks = (4LL * num_cu() + col_blocks - 1) / col_blocks;
    const long long rows = (B + chunks - 1) / chunks, least = 4 * (TPB / cw);
    const long long parts = (B + least - 1) / least;
    return {(int)(rows > least ? rows : least), (int)(parts < chunks ? parts : chunks)};
}

template <int THREADS, int PER>
hipError_t fwd(const float *mu_w, const float *var_w, const float *mu_b, const float *var_b,
               const float *mu_a, const float *var_a, float epsilon, int n, int B, float *mu_s,
               float *var_s, float *mu_z, float *var_z, hipStream_t stream) {
    // (a launch holds fewer than 2^32 threads; beyond that the workgroups walk on)
    const long long rows = TPB / THREADS, blocks = (B + rows - 1) / rows;
    const unsigned grid = (unsigned)(blocks < (1 << 22) ? blocks : 1 << 22);
    hipLaunchKernelGGL((ln_fwd_kernel<THREADS, PER>), dim3(grid), dim3(TPB), 0, stream, mu_w, var_w,
                       mu_b, var_b, mu_a, var_a, epsilon, n, B, goes_past_cache((size_t)2 * B * n),
                       mu_s, var_s, mu_z, var_z);
    return hipGetLastError();
}

}  // namespace

size_t layernorm_bwd_scratch_floats(int n, int B) {
    const int chunks = ln_chunks(n, B).most;
    return chunks == 1 ? 0 : (size_t)chunks * 4 * n;
}

hipError_t launch_layernorm_fwd(const float *mu_w, const float *var_w, const float *mu_b,
                                const float *var_b, const float *mu_a, const float *var_a,
                                float epsilon, int n, int B, float *mu_s, float *var_s,
                                float *mu_z, float *var_z, hipStream_t stream) {
    // One wave per row up to 1024 features, unless the rows would not fill the chip that way
    // (four waves for every SIMD): then a workgroup each.
    const bool many = B >= 16 * num_cu();
    auto *run = n <= 256            ? fwd<64, 1>
                : n <= 1024 && many ? fwd<64, 4>
                : n <= 1024         ? fwd<256, 1>
                : n <= 4096         ? fwd<256, 4>
                : n <= 8192         ? fwd<256, 8>
                                    : fwd<256, 0>;
    return run(mu_w, var_w, mu_b, var_b, mu_a, var_a, epsilon, n, B, mu_s, var_s, mu_z, var_z, stream);
}

hipError_t launch_layernorm_bwd(const float *mu_w, const float *var_w, const float *var_b,
                                const float *mu_a, const float *jcb, const float *mu_s,
                                const float *var_s, const float *dmu_out, const float *dvar_out,
                                float epsilon, int n, int B, int state_update, int param_update,
                                float *scratch, float *dmu, float *dvar, float *dmu_w,
                                float *dvar_w, float *dmu_b, float *dvar_b, hipStream_t stream) {
    const int rows = ln_chunks(n, B).rows, cw_log = ln_cw_log(n);
    const int chunks = (B + rows - 1) / rows, groups = (n + 3) / 4;
    const dim3 grid((groups + (1 << cw_log) - 1) >> cw_log, chunks);
    const ParamOut out = {var_w, var_b, dmu_w, dvar_w, dmu_b, dvar_b};
    hipLaunchKernelGGL(ln_bwd_kernel, grid, dim3(TPB), 0, stream, mu_w, mu_a, jcb, mu_s, var_s, dmu_out,
                       dvar_out, epsilon, n, B, rows, cw_log, state_update, param_update,
                       goes_past_cache((size_t)2 * B * n), dmu, dvar, scratch, out);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !param_update || chunks == 1) return e;
    int f_log = 0;
    while (f_log < 6 && (1 << f_log) < n) f_log++;
    hipLaunchKernelGGL(ln_bwd_final_kernel, dim3((n + (1 << f_log) - 1) >> f_log), dim3(FINAL_WAVES * 64), 0,
                       stream, scratch, n, chunks, f_log, out);
    return hipGetLastError();
}

}  // namespace tagi
