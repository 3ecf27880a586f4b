// Linear layers grouped by expert where an expert has few rows (a decoding step, a small
// batch): bound by the weights, which are streamed once per 16 (or 32) rows. gfx950.
//
// Products on v_mfma_f32_16x16x4_f32, exact fp32 products and sums: A[i][s] from lane 16 s + i,
// B[s][j] from lane 16 s + j, D[4 (l / 16) + v][l % 16] in register v of lane l. The weights
// come straight from memory in the operand's layout, the few rows of activations or
// innovations from L1 / L2; the waves of a workgroup share the reduction of an output block and are joined
// through LDS in wave order.
#include <cstdint>

#include "tagi_activation.h"
#include "tagi_grouped.h"
#include "tagi_internal.h"

namespace tagi {
namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ floatx4 mfma(float a, float b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
// Four elements at k of a row of `end`, to be passed through settle() where k + 4 > end. VEC:
// the row has four at least, and a load that would leave it is moved to end with it.
template <bool VEC>
__device__ __forceinline__ floatx4 load4(const float *row, int k, int end) {
    if (VEC) {
        const float4_any q = *reinterpret_cast<const float4_any *>(row + min(k, end - 4));
        return (floatx4){q[0], q[1], q[2], q[3]};
    }
    floatx4 v;
#pragma unroll
    for (int t = 0; t < 4; t++) v[t] = row[min(k + t, end - 1)];
    return v;
}
// What load4 brought, moved back, with zeros behind the end. (Apart from the load, so that
// loads in flight are not waited for.)
template <bool VEC>
__device__ __forceinline__ floatx4 settle(floatx4 v, int k, int end) {
    if (VEC) {
        const int n = min(max(k + 4 - end, 0), 4);
        v = n & 1 ? (floatx4){v[1], v[2], v[3], 0.f} : v;
        v = n & 2 ? (floatx4){v[2], v[3], 0.f, 0.f} : v;
        return n & 4 ? (floatx4){0.f, 0.f, 0.f, 0.f} : v;
    }
#pragma unroll
    for (int t = 0; t < 4; t++) v[t] = k + t < end ? v[t] : 0.f;
    return v;
}

// ---------------------------------------------------------------------------
// Forward, 16 outputs n of one expert. Lane (i = l % 16, s = l / 16) holds the weights
// [n0 + i][k + 4 s .. + 3] and row i's activations at the same k; component t of both meets in
// MFMA t. A wave takes every WAVES-th 32-element piece (a 128-byte line of each weight row) and
// has the next piece's loads in flight while it multiplies. Bound by the weights: 64 rows, 16
// experts of 2048 -> 4096, in 178 us back to back, 6.0 TB/s (239 us, 195 at best, where a pause
// precedes every call); one token's two of 8 experts of 4096 -> 4096 in 58 us, 4.6 TB/s.
// ---------------------------------------------------------------------------
template <int NG, bool VEC>
struct FwdPiece {
    floatx4 w0[2], w1[2], a0[NG][2], a1[NG][2];
};

template <int WAVES, int NG, bool VEC>
__device__ __forceinline__ void fwd_rows(const GroupedParams &p, int e, int n0, int r0, int end,
                                         float (*s)[8 * NG][64]) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int i = lane & 15, q = (lane >> 4) * 4, K = p.K;
    const size_t w_at = ((size_t)e * p.N + min(n0 + i, p.N - 1)) * K;
    const float *w0 = p.y0 + w_at, *w1 = p.y1 + w_at;
    // the first weights are on their way before the row indices are known
    FwdPiece<NG, VEC> x, y;
    const int step = 32 * WAVES;
    int kb = 32 * wave;
    auto load_w = [&](FwdPiece<NG, VEC> &f, int kb) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            f.w0[h] = load4<VEC>(w0, kb + 16 * h + q, K);
            f.w1[h] = load4<VEC>(w1, kb + 16 * h + q, K);
        }
    };
    if (kb < K) load_w(x, kb);
    const float *a0[NG], *a1[NG];
    bool live[NG];
#pragma unroll
    for (int g = 0; g < NG; g++) {
        int r = min(r0 + 16 * g + i, end - 1);
        live[g] = true;
        if (p.rows != nullptr) {
            r = p.rows[r];
            live[g] = (unsigned)r < (unsigned)p.T;
            if (!live[g]) r = 0;
        }
        a0[g] = p.x0 + (size_t)r * K;
        a1[g] = p.x1 + (size_t)r * K;
    }
    floatx4 acc0[NG], acc1[NG];
#pragma unroll
    for (int g = 0; g < NG; g++) acc0[g] = acc1[g] = (floatx4){0.f, 0.f, 0.f, 0.f};
    auto load_a = [&](FwdPiece<NG, VEC> &f, int kb) {
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int g = 0; g < NG; g++) {
                f.a0[g][h] = load4<VEC>(a0[g], kb + 16 * h + q, K);
                f.a1[g][h] = load4<VEC>(a1[g], kb + 16 * h + q, K);
            }
    };
    auto load = [&](FwdPiece<NG, VEC> &f, int kb) {
        load_w(f, kb);
        load_a(f, kb);
    };
    auto use = [&](FwdPiece<NG, VEC> &f, int kb) {
        if (kb + 32 > K) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int k = kb + 16 * h + q;
                f.w0[h] = settle<VEC>(f.w0[h], k, K);
                f.w1[h] = settle<VEC>(f.w1[h], k, K);
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    f.a0[g][h] = settle<VEC>(f.a0[g][h], k, K);
                    f.a1[g][h] = settle<VEC>(f.a1[g][h], k, K);
                }
            }
        }
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const float w = f.w0[h][t], v = f.w1[h][t], w2 = w * w;
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    const float m = live[g] ? f.a0[g][h][t] : 0.f, u = live[g] ? f.a1[g][h][t] : 0.f;
                    acc0[g] = mfma(w, m, acc0[g]);
                    acc1[g] = mfma(v, fmaf(m, m, u), acc1[g]);
                    acc1[g] = mfma(w2, u, acc1[g]);
                }
            }
    };
    if (kb < K) load_a(x, kb);
    for (; kb < K; kb += 2 * step) {
        if (kb + step < K) load(y, kb + step);
        use(x, kb);
        if (kb + step >= K) break;
        if (kb + 2 * step < K) load(x, kb + 2 * step);
        use(y, kb + step);
    }
    // join: s[wave][8 g + 4 a + v][lane]
#pragma unroll
    for (int g = 0; g < NG; g++)
#pragma unroll
        for (int v = 0; v < 4; v++) {
            s[wave][8 * g + v][lane] = acc0[g][v];
            s[wave][8 * g + 4 + v][lane] = acc1[g][v];
        }
    __syncthreads();
    // thread: output n0 + x of row j of group g
#pragma unroll
    for (int at = tid; at < 256 * NG; at += WAVES * 64) {
        const int g = at >> 8, j = (at >> 4) & 15, x16 = at & 15;
        const int l = (x16 >> 2) * 16 + j, v = x16 & 3;
        float m = 0.f, u = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            m += s[w][8 * g + v][l];
            u += s[w][8 * g + 4 + v][l];
        }
        const int r = r0 + 16 * g + j, n = n0 + x16;
        if (r < end && n < p.N) {
            if (p.e0 != nullptr) {
                m += p.e0[(size_t)e * p.N + n];
                u += p.e1[(size_t)e * p.N + n];
            }
            store_activated(p.act, m, u, (size_t)r * p.N + n, p.out0, p.out1, p.out2);
        }
    }
    __syncthreads();
}

template <int WAVES, int NG, bool VEC>
__global__ __launch_bounds__(WAVES * 64, NG == 1 && VEC ? 4 : 2) void rows_fwd_kernel(GroupedParams p) {
    __shared__ float s[WAVES][8 * NG][64];
    const int blocks = (p.N + 15) / 16, slot = blockIdx.x / blocks, n0 = (blockIdx.x - slot * blocks) * 16;
    int r0, end;
    const int e = find_rows(p.offsets, p.E, p.R, 16 * NG, slot, r0, end);
    if (e >= 0) fwd_rows<WAVES, NG, VEC>(p, e, n0, r0, end, s);
}

// ---------------------------------------------------------------------------
// State backward, 16 C inputs k of one expert (C = 4, or 1 where few inputs and rows would leave
// most of the chip idle). Lane (i, s) holds mu_w[n + 4 s + u][k0 + C i .. + C - 1] for u = 0..3
// (C = 4: a load covers four weight rows of 256 bytes) and row i's innovations at n + 4 s .. + 3:
// component t of step u meets component u of the innovations in an MFMA of its own sum,
// D[i][j] = output k0 + C i + t of row j. Bound by the weights, beyond some ten rows per expert
// by the matrix instructions: 192 rows, 8 experts of 2048 -> 4096, in 83 us, 3.2 TB/s.
// ---------------------------------------------------------------------------
template <int NG, int C>
struct DzPiece {
    float w[4][C];
    floatx4 d0[NG], d1[NG];
};

template <int WAVES, int NG, int C, bool VEC>
__device__ __forceinline__ void dz_rows(const GroupedParams &p, int e, int k0, int r0, int end,
                                        float (*s)[4 * C][65]) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int i = lane & 15, q = (lane >> 4) * 4, K = p.K, N = p.N;
    const float *w = p.y0 + (size_t)e * N * K;
    const int k = k0 + C * i;
    const float *d0[NG], *d1[NG];
#pragma unroll
    for (int g = 0; g < NG; g++) {
        const size_t r = (size_t)min(r0 + 16 * g + i, end - 1) * N;
        d0[g] = p.x0 + r;
        d1[g] = p.x1 + r;
    }
    floatx4 acc0[NG][C], acc1[NG][C];
#pragma unroll
    for (int g = 0; g < NG; g++)
#pragma unroll
        for (int t = 0; t < C; t++) acc0[g][t] = acc1[g][t] = (floatx4){0.f, 0.f, 0.f, 0.f};
    auto load = [&](DzPiece<NG, C> &f, int nb) {
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const float *row = w + (size_t)min(nb + q + u, N - 1) * K;
            if constexpr (C == 4) {
                const floatx4 x = load4<VEC>(row, k, K);
#pragma unroll
                for (int t = 0; t < C; t++) f.w[u][t] = x[t];
            } else {
                f.w[u][0] = row[min(k, K - 1)];   // (columns beyond the last are not stored)
            }
        }
#pragma unroll
        for (int g = 0; g < NG; g++) {
            f.d0[g] = load4<VEC>(d0[g], nb + q, N);
            f.d1[g] = load4<VEC>(d1[g], nb + q, N);
        }
    };
    const bool edge = C == 4 && k0 + 64 > K;
    auto use = [&](DzPiece<NG, C> &f, int nb) {
        if (edge || nb + 16 > N) {
#pragma unroll
            for (int u = 0; u < 4; u++) {
                if constexpr (C == 4) {
                    const floatx4 x = settle<VEC>((floatx4){f.w[u][0], f.w[u][1], f.w[u][2], f.w[u][3]}, k, K);
#pragma unroll
                    for (int t = 0; t < C; t++) f.w[u][t] = x[t];
                }
#pragma unroll
                for (int t = 0; t < C; t++)
                    if (nb + q + u >= N) f.w[u][t] = 0.f;
            }
#pragma unroll
            for (int g = 0; g < NG; g++) {
                f.d0[g] = settle<VEC>(f.d0[g], nb + q, N);
                f.d1[g] = settle<VEC>(f.d1[g], nb + q, N);
            }
        }
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int t = 0; t < C; t++) {
                const float x = f.w[u][t], x2 = x * x;
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    acc0[g][t] = mfma(x, f.d0[g][u], acc0[g][t]);
                    acc1[g][t] = mfma(x2, f.d1[g][u], acc1[g][t]);
                }
            }
    };
    DzPiece<NG, C> x, y;
    const int step = 16 * WAVES;
    int nb = 16 * wave;
    if (nb < N) load(x, nb);
    for (; nb < N; nb += 2 * step) {
        if (nb + step < N) load(y, nb + step);
        use(x, nb);
        if (nb + step >= N) break;
        if (nb + 2 * step < N) load(x, nb + 2 * step);
        use(y, nb + step);
    }
    constexpr int COLS = 16 * C, THREADS = WAVES * 64;
    constexpr int STEPS = (16 * COLS + THREADS - 1) / THREADS;   // outputs of a thread
#pragma unroll
    for (int g = 0; g < NG; g++) {
        float sum[2][STEPS];
#pragma unroll
        for (int a = 0; a < 2; a++) {
            __syncthreads();
#pragma unroll
            for (int t = 0; t < C; t++)
#pragma unroll
                for (int v = 0; v < 4; v++) s[wave][4 * t + v][lane] = (a == 0 ? acc0 : acc1)[g][t][v];
            __syncthreads();
#pragma unroll
            for (int h = 0; h < STEPS; h++) {
                const int c = tid % COLS, j = (tid / COLS + THREADS / COLS * h) & 15, at = c / C;
                const int l = (at >> 2) * 16 + j, x = 4 * (c % C) + (at & 3);
                float m = 0.f;
#pragma unroll
                for (int w = 0; w < WAVES; w++) m += s[w][x][l];
                sum[a][h] = m;
            }
        }
#pragma unroll
        for (int h = 0; h < STEPS; h++) {
            const int c = k0 + tid % COLS, j = tid / COLS + THREADS / COLS * h, r = r0 + 16 * g + j;
            if (j < 16 && r < end && c < K) {
                const size_t at = (size_t)r * K + c;
                const float f = p.e0 != nullptr ? p.e0[at] : 1.f;
                p.out0[at] = sum[0][h] * f;
                p.out1[at] = sum[1][h] * f * f;
            }
        }
    }
    __syncthreads();
}

template <int WAVES, int NG, int C, bool VEC>
__global__ __launch_bounds__(WAVES * 64, WAVES == 8 && NG == 1 && VEC ? 4 : 2) void rows_dz_kernel(GroupedParams p) {
    __shared__ float s[WAVES][4 * C][65];
    const int blocks = (p.K + 16 * C - 1) / (16 * C), slot = blockIdx.x / blocks;
    const int k0 = (blockIdx.x - slot * blocks) * 16 * C;
    int r0, end;
    const int e = find_rows(p.offsets, p.E, p.R, 16 * NG, slot, r0, end);
    if (e >= 0) dz_rows<WAVES, NG, C, VEC>(p, e, k0, r0, end, s);
}

// ---------------------------------------------------------------------------
// Weight (and bias) backward: a wave owns eight rows n by 256 columns k of one expert's
// weights, four columns per lane, and adds the outer products of the expert's rows four at a
// time; the innovations of a row are the same for the whole wave. Twelve bytes move per
// weight, two multiplications-and-additions per row of the batch: bound by memory up to some
// tens of rows.
// ---------------------------------------------------------------------------
constexpr int DW_ROWS = 8, DW_COLS = 256, DW_WAVES = 4;

template <bool VEC>
__global__ __launch_bounds__(DW_WAVES * 64) void rows_dw_kernel(GroupedParams p) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int K = p.K, N = p.N;
    const int col_blocks = (K + DW_COLS - 1) / DW_COLS;
    const int row_blocks = (N + DW_ROWS * DW_WAVES - 1) / (DW_ROWS * DW_WAVES);
    const int kb = blockIdx.x % col_blocks, rest = blockIdx.x / col_blocks;
    const int e = rest / row_blocks;
    const int n0 = (rest - e * row_blocks) * DW_ROWS * DW_WAVES + wave * DW_ROWS;
    const int k = kb * DW_COLS + lane * 4;
    int first, end;
    group_rows(p.offsets, e, p.R, first, end);
    if (n0 >= N) return;
    const int rows_n = min(DW_ROWS, N - n0);
    const float *__restrict__ d0 = p.x0, *__restrict__ d1 = p.x1;
    // the factors of the result are on their way first
    floatx4 w[DW_ROWS];
#pragma unroll
    for (int n = 0; n < DW_ROWS; n++)
        w[n] = load4<VEC>(p.e0 + ((size_t)e * N + n0 + min(n, rows_n - 1)) * K, min(k, K - 1), K);
    if (p.db0 != nullptr && kb == 0) {   // lane: row n0 + lane % 8, every eighth row of the batch
        float m = 0.f, v = 0.f;
        const int n = n0 + min(lane & 7, rows_n - 1);
        for (int r = first + (lane >> 3); r < end; r += 8) {
            m += d0[(size_t)r * N + n];
            v += d1[(size_t)r * N + n];
        }
#pragma unroll
        for (int off = 8; off < 64; off <<= 1) {
            m += __shfl_xor(m, off, 64);
            v += __shfl_xor(v, off, 64);
        }
        if (lane < rows_n) {
            const size_t at = (size_t)e * N + n0 + lane;
            const float vb = p.e1[at];
            p.db0[at] = vb * m;
            p.db1[at] = vb * vb * v;
        }
    }
    if (k >= K) return;
    floatx4 acc0[DW_ROWS], acc1[DW_ROWS];
#pragma unroll
    for (int n = 0; n < DW_ROWS; n++) acc0[n] = acc1[n] = (floatx4){0.f, 0.f, 0.f, 0.f};
    for (int r = first; r < end; r += 4) {
        floatx4 a[4], a2[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            int s = min(r + j, end - 1);
            bool live = r + j < end;
            if (p.rows != nullptr) {
                s = p.rows[s];
                live = live && (unsigned)s < (unsigned)p.T;
                if (!live) s = 0;
            }
            a[j] = settle<VEC>(load4<VEC>(p.y0 + (size_t)s * K, k, K), k, K);
            if (!live) a[j] = (floatx4){0.f, 0.f, 0.f, 0.f};
            a2[j] = a[j] * a[j];
        }
#pragma unroll
        for (int n = 0; n < DW_ROWS; n++) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const size_t at = (size_t)min(r + j, end - 1) * N + min(n0 + n, N - 1);
                const bool live = r + j < end;
                const float m = live ? d0[at] : 0.f, v = live ? d1[at] : 0.f;
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    acc0[n][c] = fmaf(m, a[j][c], acc0[n][c]);
                    acc1[n][c] = fmaf(v, a2[j][c], acc1[n][c]);
                }
            }
        }
    }
#pragma unroll
    for (int n = 0; n < DW_ROWS; n++) {
        if (n >= rows_n) break;
        const size_t at = ((size_t)e * N + n0 + n) * K + k;
        const floatx4 f = settle<VEC>(w[n], k, K);
        float4_any m, v;
#pragma unroll
        for (int c = 0; c < 4; c++) {
            m[c] = acc0[n][c] * f[c];
            v[c] = acc1[n][c] * f[c] * f[c];
        }
        if (k + 4 <= K) {
            *reinterpret_cast<float4_any *>(p.out0 + at) = m;
            *reinterpret_cast<float4_any *>(p.out1 + at) = v;
        } else {
#pragma unroll
            for (int c = 0; c < 3; c++)
                if (k + c < K) {
                    p.out0[at + c] = m[c];
                    p.out1[at + c] = v[c];
                }
        }
    }
}

template <int WAVES, int NG, bool VEC>
void rows_fwd(const GroupedParams &p, unsigned grid, hipStream_t stream) {
    hipLaunchKernelGGL((rows_fwd_kernel<WAVES, NG, VEC>), dim3(grid), dim3(WAVES * 64), 0, stream, p);
}
template <int WAVES, int NG, int C, bool VEC>
void rows_dz(const GroupedParams &p, unsigned slots, hipStream_t stream) {
    const unsigned blocks = (p.K + 16 * C - 1) / (16 * C);
    hipLaunchKernelGGL((rows_dz_kernel<WAVES, NG, C, VEC>), dim3(blocks * slots), dim3(WAVES * 64), 0, stream, p);
}

}  // namespace

hipError_t launch_grouped_rows(GroupedMode mode, const GroupedParams &p, bool vec, hipStream_t stream) {
    // experts that can have rows
    const int used = p.E < p.R ? p.E : p.R;
    // Two groups of sixteen rows share a pass over the weights where experts have more than
    // eight rows on average; one group leaves registers for twice the waves, which is also
    // better where the forward's blocks are few (two groups / one: 87 rows, 3 experts of 3878
    // -> 37: 37 / 24 us; 40 rows, 2 experts of 4096 -> 512: 43 / 33; 777 rows, 6 experts of 301
    // -> 200: 12 / 17).
    const bool one = (long long)p.R <= 8LL * p.E ||
                     (mode == GROUPED_FWD && (p.R / 16 + used) * ((p.N + 15LL) / 16) <= 256);
    const unsigned slots = p.R / (one ? 16 : 32) + used;   // groups of rows at most
    if (mode == GROUPED_FWD) {
        const unsigned blocks = (p.N + 15) / 16, grid = blocks * slots;
        // Waves that share a block: many blocks fill the chip with few waves each, which
        // spend less of their time starting and joining. 4 / 8 / 16 waves: 216 / 231 / 266 us
        // at 16 x 256 blocks of 2048, 73 / 61 / 69 at 2 x 256 of 4096, 43 / 30 / 26 at 2 x 64.
        const long long working = (long long)used * blocks;
        if (!vec)
            one ? rows_fwd<8, 1, false>(p, grid, stream) : rows_fwd<8, 2, false>(p, grid, stream);
        // (a wave needs some 32-element pieces to be worth its join. 32 rows: 4 / 8 waves 177 /
        // 221 us at 8 x 256 blocks of 2048, 59 / 76 at 16 x 64 of 1024, 28 / 28 at 2 x 128 of
        // 2048, 48 / 43 at 2 x 32 of 4096)
        else if (!one)
            p.K <= 512 || working > 256 ? rows_fwd<4, 2, true>(p, grid, stream)
                                        : rows_fwd<8, 2, true>(p, grid, stream);
        else if (working > 1024)
            rows_fwd<4, 1, true>(p, grid, stream);
        else if (working > 256)
            rows_fwd<8, 1, true>(p, grid, stream);
        else
            rows_fwd<16, 1, true>(p, grid, stream);
    } else if (mode == GROUPED_DZ) {
        // Blocks of 16 inputs, by sixteen waves, while those of 64 are too few: wide / narrow
        // for blocks of 64 inputs x groups of rows, N = 2048, one row per expert 4: 27 / 13,
        // 64: 32 / 15, 128: 32 / 21, 256: 33 / 31 us; twelve rows 4: 38 / 18, 128: 41 / 39,
        // 256: 43 / 74 us.
        const long long groups = p.R / 32 + used / 2;
        const bool narrow = (groups > used ? groups : used) * ((p.K + 63) / 64) <= 128;
        if (!vec)
            one ? rows_dz<8, 1, 4, false>(p, slots, stream) : rows_dz<8, 2, 4, false>(p, slots, stream);
        else if (narrow)
            one ? rows_dz<16, 1, 1, true>(p, slots, stream) : rows_dz<16, 2, 1, true>(p, slots, stream);
        else
            one ? rows_dz<8, 1, 4, true>(p, slots, stream) : rows_dz<8, 2, 4, true>(p, slots, stream);
    } else {
        const int rows = DW_ROWS * DW_WAVES;
        const dim3 grid((unsigned)((p.K + DW_COLS - 1) / DW_COLS) * ((p.N + rows - 1) / rows) * p.E);
        if (vec)
            hipLaunchKernelGGL(rows_dw_kernel<true>, grid, dim3(DW_WAVES * 64), 0, stream, p);
        else
            hipLaunchKernelGGL(rows_dw_kernel<false>, grid, dim3(DW_WAVES * 64), 0, stream, p);
    }
    return hipGetLastError();
}

}  // namespace tagi
