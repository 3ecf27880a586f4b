// Linear layers grouped by expert: row r of expert e (offsets[e] <= r < offsets[e+1])
// meets the weights [e][N][K]. gfx950.
#include <cstdint>

#include "tagi_activation.h"
#include "tagi_internal.h"

namespace tagi {
namespace {

constexpr int TPB = 256;
constexpr int BT = 64;    // rows and columns of a workgroup's tile
constexpr int KT = 16;

// Rows [first, end) of expert e, whatever the offsets hold: inside 0..R, never negative.
__device__ __forceinline__ void group_rows(const int *__restrict__ offsets, int e, int R, int &first,
                                           int &end) {
    first = min(max(offsets[e], 0), R);
    end = min(max(offsets[e + 1], first), R);
}

// The tile_at-th tile of `rows` rows over all groups: its expert, or -1 beyond the last.
__device__ __forceinline__ int find_tile(const int *__restrict__ offsets, int E, int R, int tile_at,
                                         int rows, int &r0, int &end) {
    for (int e = 0; e < E; e++) {
        int first;
        group_rows(offsets, e, R, first, end);
        const int tiles = (end - first + rows - 1) / rows;
        if (tile_at < tiles) {
            r0 = first + tile_at * rows;
            return e;
        }
        tile_at -= tiles;
    }
    return -1;
}

// One 64 x 64 tile of an output pair. FWD: rows r, columns n, sum over k. DZ: rows r,
// columns k, sum over n. DW: rows n, columns k, sum over the expert's rows r.
template <int MODE>
__global__ __launch_bounds__(TPB) void grouped_simple_kernel(GroupedParams p) {
    __shared__ float x0[KT][BT], x1[KT][BT], y0[KT][BT], y1[KT][BT];
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    int e, r0 = 0, end = 0, m0;
    const int col_tiles = ((MODE == GROUPED_FWD ? p.N : p.K) + BT - 1) / BT;
    const int ct = blockIdx.x % col_tiles, rt = blockIdx.x / col_tiles;
    if (MODE == GROUPED_DW) {
        const int n_tiles = (p.N + BT - 1) / BT;
        e = rt / n_tiles;
        group_rows(p.offsets, e, p.R, r0, end);
        m0 = rt % n_tiles * BT;
    } else {
        e = find_tile(p.offsets, p.E, p.R, rt, BT, r0, end);
        if (e < 0) return;
        m0 = r0;
    }
    const int c0 = ct * BT;
    const int M = MODE == GROUPED_DW ? p.N : end;
    const int C = MODE == GROUPED_FWD ? p.N : p.K;
    const int S = MODE == GROUPED_FWD ? p.K : MODE == GROUPED_DZ ? p.N : end - r0;
    const size_t w_at = (size_t)e * p.N * p.K;
    float a0[4][4] = {}, a1[4][4] = {};
    auto source = [&](int r) {
        if (p.rows == nullptr) return r;
        const int s = p.rows[r];
        return (unsigned)s < (unsigned)p.T ? s : -1;
    };
    for (int k0 = 0; k0 < S; k0 += KT) {
        for (int i = tid; i < BT * KT; i += TPB) {
            const int m = MODE == GROUPED_DW ? i % BT : i / KT, k = MODE == GROUPED_DW ? i / BT : i % KT;
            float u0 = 0.f, u1 = 0.f;
            if (m0 + m < M && k0 + k < S) {
                if (MODE == GROUPED_FWD) {
                    const int s = source(m0 + m);
                    if (s >= 0) {
                        u0 = p.x0[(size_t)s * p.K + k0 + k];
                        u1 = p.x1[(size_t)s * p.K + k0 + k];
                    }
                } else {
                    const size_t at = MODE == GROUPED_DZ ? (size_t)(m0 + m) * p.N + k0 + k
                                                         : (size_t)(r0 + k0 + k) * p.N + m0 + m;
                    u0 = p.x0[at];
                    u1 = p.x1[at];
                }
            }
            x0[k][m] = u0;
            x1[k][m] = u1;
            const int c = MODE == GROUPED_FWD ? i / KT : i % BT, ck = MODE == GROUPED_FWD ? i % KT : i / BT;
            float v0 = 0.f, v1 = 0.f;
            if (c0 + c < C && k0 + ck < S) {
                if (MODE == GROUPED_FWD) {
                    v0 = p.y0[w_at + (size_t)(c0 + c) * p.K + k0 + ck];
                    v1 = p.y1[w_at + (size_t)(c0 + c) * p.K + k0 + ck];
                } else if (MODE == GROUPED_DZ) {
                    v0 = p.y0[w_at + (size_t)(k0 + ck) * p.K + c0 + c];
                } else {
                    const int s = source(r0 + k0 + ck);
                    if (s >= 0) v0 = p.y0[(size_t)s * p.K + c0 + c];
                }
            }
            y0[ck][c] = v0;
            y1[ck][c] = v1;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < KT; k++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float u0 = x0[k][ty * 4 + i], u1 = x1[k][ty * 4 + i];
                    const float v0 = y0[k][tx * 4 + j], v1 = y1[k][tx * 4 + j];
                    a0[i][j] += u0 * v0;
                    if (MODE == GROUPED_FWD)
                        a1[i][j] += (u1 + u0 * u0) * v1 + u1 * (v0 * v0);
                    else
                        a1[i][j] += u1 * (v0 * v0);
                }
        __syncthreads();
    }
    for (int i = 0; i < 4; i++)
        for (int j = 0; j < 4; j++) {
            const int m = m0 + ty * 4 + i, c = c0 + tx * 4 + j;
            if (m >= M || c >= C) continue;
            float s0 = a0[i][j], s1 = a1[i][j];
            if (MODE == GROUPED_FWD) {
                if (p.e0 != nullptr) {
                    s0 += p.e0[(size_t)e * p.N + c];
                    s1 += p.e1[(size_t)e * p.N + c];
                }
                store_activated(p.act, s0, s1, (size_t)m * p.N + c, p.out0, p.out1, p.out2);
            } else {
                const size_t at = MODE == GROUPED_DZ ? (size_t)m * p.K + c : w_at + (size_t)m * p.K + c;
                const float f = p.e0 != nullptr ? p.e0[at] : 1.f;
                p.out0[at] = s0 * f;
                p.out1[at] = s1 * f * f;
            }
        }
}

// Bias innovations of one expert's 64 columns: four waves take every fourth row.
__global__ __launch_bounds__(TPB) void grouped_db_kernel(GroupedParams p) {
    __shared__ float s[2][TPB];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n = blockIdx.x * 64 + lane, e = blockIdx.y;
    int first, end;
    group_rows(p.offsets, e, p.R, first, end);
    float m = 0.f, v = 0.f;
    if (n < p.N)
        for (int r = first + wave; r < end; r += 4) {
            m += p.x0[(size_t)r * p.N + n];
            v += p.x1[(size_t)r * p.N + n];
        }
    s[0][threadIdx.x] = m;
    s[1][threadIdx.x] = v;
    __syncthreads();
    if (wave != 0 || n >= p.N) return;
    m = (s[0][lane] + s[0][64 + lane]) + (s[0][128 + lane] + s[0][192 + lane]);
    v = (s[1][lane] + s[1][64 + lane]) + (s[1][128 + lane] + s[1][192 + lane]);
    const size_t at = (size_t)e * p.N + n;
    const float vb = p.e0[at];
    p.out0[at] = vb * m;
    p.out1[at] = vb * vb * v;
}

inline int ceil_div(int a, int b) { return (a + b - 1) / b; }

}  // namespace

hipError_t launch_grouped(GroupedMode mode, const GroupedParams &p, hipStream_t stream) {
    // row tiles over all groups: every group ends with at most one part tile
    const unsigned row_tiles = p.R / BT + (p.E < p.R ? p.E : p.R);
    if (mode == GROUPED_FWD)
        hipLaunchKernelGGL(grouped_simple_kernel<GROUPED_FWD>, dim3(ceil_div(p.N, BT) * row_tiles),
                           dim3(TPB), 0, stream, p);
    else if (mode == GROUPED_DZ)
        hipLaunchKernelGGL(grouped_simple_kernel<GROUPED_DZ>, dim3(ceil_div(p.K, BT) * row_tiles),
                           dim3(TPB), 0, stream, p);
    else
        hipLaunchKernelGGL(grouped_simple_kernel<GROUPED_DW>,
                           dim3((unsigned)ceil_div(p.K, BT) * ceil_div(p.N, BT) * p.E), dim3(TPB), 0,
                           stream, p);
    return hipGetLastError();
}

hipError_t launch_grouped_db(const GroupedParams &p, hipStream_t stream) {
    hipLaunchKernelGGL(grouped_db_kernel, dim3(ceil_div(p.N, 64), p.E), dim3(TPB), 0, stream, p);
    return hipGetLastError();
}

}  // namespace tagi
