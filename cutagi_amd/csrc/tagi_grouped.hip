// Linear layers grouped by expert: row r of expert e (offsets[e] <= r < offsets[e+1])
// meets the weights [e][N][K]. gfx950.
#include <cstdint>

#include "tagi_activation.h"
#include "tagi_internal.h"

namespace tagi {
namespace {

constexpr int TPB = 256;
constexpr int MAX_GROUPS = 1024;

// Rows [first, end) of expert e, whatever the offsets hold: inside 0..R, never negative.
__device__ __forceinline__ void group_rows(const int *__restrict__ offsets, int e, int R, int &first,
                                           int &end) {
    first = min(max(offsets[e], 0), R);
    end = min(max(offsets[e + 1], first), R);
}

// ---------------------------------------------------------------------------
// Tiled kernel. fp32 products on the bf16 matrix instructions.
//
// x = h + m + l with h, m, l in bf16 (each the rounding of what the ones before it leave
// out): |x - h| <= 2^-9 |x|, |x - h - m| <= 2^-18 |x|, |x - h - m - l| <= 2^-27 |x|, and bf16 has
// fp32's range, so no scaling is needed. Of the nine products of two such numbers
//     x y ~ hh + hm + mh + mm + hl + lh
// are formed; what is left out (ml, lm, ll and the residues) is below 2^-25 |x y|, half of
// fp32's own half step. Products of two bf16 are exact in the fp32 accumulator. Six
// instructions at 16 times the fp32 matrix rate leave 2.7 times that rate.
// An infinity (or a magnitude beyond bf16's 3.39e38) has the residue NaN and gives NaN, where
// fp32 arithmetic would give an infinity or NaN.
//
// A workgroup owns 128 x 128 tiles of an output pair and walks them one after the other. Four
// of its waves load the operands, form the sums and squares that the variance needs, split
// them and write the pieces to LDS; the other four read fragments and issue matrix
// instructions on 64 x 64 sub-tiles. Every SIMD holds one wave of each kind, so the vector
// work of the split runs under the matrix instructions without any interleaving in the code,
// and an element is split once for the four or two waves that read it. Two LDS stages of 16
// reduction elements, one barrier per stage.
// ---------------------------------------------------------------------------
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef float floatx16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ unsigned pack_bf16(float a, float b) {
    const bf16x2 r = __builtin_convertvector((floatx2){a, b}, bf16x2);
    return __builtin_bit_cast(unsigned, r);
}
// the three bf16 pieces of a and b, packed pairwise
__device__ __forceinline__ void split_pair(float a, float b, unsigned (&piece)[3]) {
#pragma unroll
    for (int s = 0; s < 3; s++) {
        piece[s] = pack_bf16(a, b);
        if (s < 2) {
            a -= __uint_as_float(piece[s] << 16);
            b -= __uint_as_float(piece[s] & 0xffff0000u);
        }
    }
}

constexpr int TM = 128;             // rows and columns of a tile
constexpr int TK = 16;              // reduction elements of a stage
constexpr int TILE_THREADS = 512;   // 256 that stage, 256 that multiply
// An LDS plane holds eight reduction elements (16 bytes) of the tile's 128 rows (or columns)
// for one piece of one operand. The 128 bytes between planes put the two planes of a
// 16-element stage on different banks when four lanes write one row.
constexpr int PLANE = TM * 16 + 128;

template <int MODE>
struct TileShape {
    static constexpr int OPS = MODE == GROUPED_FWD ? 3 : 2;         // operands per side
    static constexpr int SIDE = OPS * 3 * 2 * PLANE;
    static constexpr int STAGE = 2 * SIDE;
    static constexpr int LDS = 2 * STAGE + (MAX_GROUPS + 1) * 4;
    // reduction contiguous in memory on the row / column side?
    static constexpr bool AK = MODE != GROUPED_DW, BK = MODE == GROUPED_FWD;
};

// Where row (or column) m of a tile sits in its planes. Operands whose reduction index is
// the slow one are loaded four neighbouring columns at a time; they go to positions 32 apart,
// so that neighbouring lanes write neighbouring 16-byte places.
template <bool KCONTIG>
__device__ __forceinline__ int row_at(int pos) {
    return KCONTIG ? pos : (pos & 31) * 4 + (pos >> 5);
}

// Four elements of a row that starts at `base` (16-byte aligned groups), or guarded ones.
template <bool VEC>
__device__ __forceinline__ float4 load4(const float *base, int k, int end) {
    if (VEC) return *reinterpret_cast<const float4 *>(base + min(k, end - 4));
    float4 v;
    v.x = base[min(k, end - 1)];
    v.y = base[min(k + 1, end - 1)];
    v.z = base[min(k + 2, end - 1)];
    v.w = base[min(k + 3, end - 1)];
    return v;
}
__device__ __forceinline__ float4 keep4(float4 v, int k, int end) {
    v.x = k < end ? v.x : 0.f;
    v.y = k + 1 < end ? v.y : 0.f;
    v.z = k + 2 < end ? v.z : 0.f;
    v.w = k + 3 < end ? v.w : 0.f;
    return v;
}

__device__ __forceinline__ void stage_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// The operands of one side from the values loaded: FWD rows (mu_a, var_a + mu_a^2, var_a),
// FWD columns (mu_w, var_w, mu_w^2), innovations (delta_mu, delta_var), DZ / DW columns
// (w or a, its square).
template <int MODE, bool ROWS>
__device__ __forceinline__ void operands(float u, float v, float (&o)[3]) {
    o[0] = u;
    if (MODE == GROUPED_FWD) {
        o[1] = ROWS ? fmaf(u, u, v) : v;
        o[2] = ROWS ? v : u * u;
    } else {
        o[1] = ROWS ? v : u * u;
    }
}

// A tile of the problem: expert, first row / column, reduction range, and the rows that exist.
struct Tile {
    int e, m0, c0;      // expert, first output row, first output column
    int m_end, c_end;   // one past the last
    int r0, red;        // DW: first row of the expert; length of the reduction
};

// Side with its reduction index contiguous: thread u of 128 holds elements 4 (u % 4) .. + 3
// of the stage for the rows u / 4 + 32 i.
template <int MODE, bool ROWS, bool VEC>
struct StageK {
    const float *p0[4], *p1[4];
    bool live[4];
    float4 v0[4], v1[4];
    int k, red;
    __device__ __forceinline__ void start(const GroupedParams &p, const Tile &t, int u) {
        k = (u & 3) * 4;
        red = t.red;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int row = (u >> 2) + 32 * i;
            live[i] = true;
            size_t at;
            if (ROWS) {
                const int m = min(t.m0 + row, t.m_end - 1);
                int s = m;
                if (MODE == GROUPED_FWD && p.rows != nullptr) {
                    s = p.rows[m];
                    live[i] = (unsigned)s < (unsigned)p.T;
                    if (!live[i]) s = 0;
                }
                at = (size_t)s * t.red;
            } else {
                at = ((size_t)t.e * p.N + min(t.c0 + row, t.c_end - 1)) * t.red;
            }
            p0[i] = (ROWS ? p.x0 : p.y0) + at;
            p1[i] = (ROWS ? p.x1 : p.y1) + at;
        }
    }
    __device__ __forceinline__ void load(int stage) {
        const int at = stage * TK + k;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v0[i] = load4<VEC>(p0[i], at, red);
            v1[i] = load4<VEC>(p1[i], at, red);
        }
    }
    __device__ __forceinline__ void write(char *side, int stage, int u) const {
        const int at = stage * TK + k;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float4 a = keep4(v0[i], live[i] ? at : red, red);
            const float4 b = keep4(v1[i], live[i] ? at : red, red);
            float x[4][3];
            operands<MODE, ROWS>(a.x, b.x, x[0]);
            operands<MODE, ROWS>(a.y, b.y, x[1]);
            operands<MODE, ROWS>(a.z, b.z, x[2]);
            operands<MODE, ROWS>(a.w, b.w, x[3]);
            char *to = side + ((u & 3) >> 1) * PLANE + ((u >> 2) + 32 * i) * 16 + (u & 1) * 8;
#pragma unroll
            for (int o = 0; o < TileShape<MODE>::OPS; o++) {
                unsigned lo[3], hi[3];
                split_pair(x[0][o], x[1][o], lo);
                split_pair(x[2][o], x[3][o], hi);
#pragma unroll
                for (int s = 0; s < 3; s++)
                    *reinterpret_cast<uint2 *>(to + (o * 3 + s) * 2 * PLANE) = make_uint2(lo[s], hi[s]);
            }
        }
    }
};

// Side with its reduction index slow: thread u of 128 holds the columns 4 c .. + 3 for the
// reduction elements 4 g .. + 3, g = 2 (u / 64) + u % 2, c = (u % 64) / 2.
template <int MODE, bool ROWS, bool VEC>
struct StageM {
    const float *q0, *q1;     // element (reduction 0, column 0) of the operand
    int ld, first, red, r0, g;
    int col, cols;            // column of the thread, columns that exist
    const int *rows;
    int tokens;
    float4 v0[4], v1[4];
    bool live[4];
    __device__ __forceinline__ void start(const GroupedParams &p, const Tile &t, int u) {
        g = 2 * (u >> 6) + (u & 1);
        red = t.red;
        r0 = t.r0;
        rows = nullptr;
        tokens = 0;
        if (ROWS) {             // DW: innovations [R][N], columns n
            ld = p.N;
            q0 = p.x0 + (size_t)t.r0 * p.N;
            q1 = p.x1 + (size_t)t.r0 * p.N;
            first = t.m0;
            cols = t.m_end;
        } else {
            ld = p.K;
            first = t.c0;
            cols = t.c_end;
            if (MODE == GROUPED_DZ) {
                q0 = p.y0 + (size_t)t.e * p.N * p.K;
            } else {            // DW: activations [T or R][K]
                rows = p.rows;
                tokens = p.T;
                q0 = p.y0 + (rows == nullptr ? (size_t)t.r0 * p.K : 0);
            }
            q1 = q0;
        }
        col = first + ((u & 63) >> 1) * 4;
    }
    __device__ __forceinline__ void load(int stage) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = min(stage * TK + 4 * g + i, red - 1);
            size_t s = (size_t)r;
            live[i] = true;
            if (!ROWS && MODE == GROUPED_DW && rows != nullptr) {
                const int token = rows[r0 + r];
                live[i] = (unsigned)token < (unsigned)tokens;
                s = live[i] ? token : 0;
            }
            // (columns beyond the last are computed and not stored; they only have to be
            // addresses that exist)
            v0[i] = load4<VEC>(q0 + s * ld, col, cols);
            if (ROWS) v1[i] = load4<VEC>(q1 + s * ld, col, cols);
        }
    }
    __device__ __forceinline__ void write(char *side, int stage, int u) const {
        const int c = (u & 63) >> 1;
        float a[4][4], b[4][4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const bool in = live[i] && stage * TK + 4 * g + i < red;
            a[i][0] = in ? v0[i].x : 0.f;
            a[i][1] = in ? v0[i].y : 0.f;
            a[i][2] = in ? v0[i].z : 0.f;
            a[i][3] = in ? v0[i].w : 0.f;
            if (ROWS) {
                b[i][0] = in ? v1[i].x : 0.f;
                b[i][1] = in ? v1[i].y : 0.f;
                b[i][2] = in ? v1[i].z : 0.f;
                b[i][3] = in ? v1[i].w : 0.f;
            }
        }
        char *to = side + (g >> 1) * PLANE + c * 16 + (g & 1) * 8;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float x[4][3];
#pragma unroll
            for (int i = 0; i < 4; i++) operands<MODE, ROWS>(a[i][j], ROWS ? b[i][j] : 0.f, x[i]);
#pragma unroll
            for (int o = 0; o < 2; o++) {
                unsigned lo[3], hi[3];
                split_pair(x[0][o], x[1][o], lo);
                split_pair(x[2][o], x[3][o], hi);
#pragma unroll
                for (int s = 0; s < 3; s++)
                    *reinterpret_cast<uint2 *>(to + (o * 3 + s) * 2 * PLANE + j * 32 * 16) =
                        make_uint2(lo[s], hi[s]);
            }
        }
    }
};

// The tiles of a workgroup: XCD x (workgroups x, x + 8, ...) takes the x-th eighth of the tile
// list, its workgroups every (workgroups of the XCD)-th tile of that.
//   FWD, DZ: row tiles over all groups, eight of them by all columns, so that the workgroups
//            of an XCD share rows and columns in its L2
//   DW: the same eighth of every expert's tiles, whatever its number of rows; an eighth of
//            all experts' tiles in order where an expert has too few to divide
template <int MODE>
struct TileList {
    int tiles_m, tiles_c, lo, count;   // this XCD's part of the list
    int per;                           // DW: tiles of it per expert, 0: a part of all tiles in order
    const int *prefix;                 // row tiles before every group (LDS)
    __device__ __forceinline__ bool get(const GroupedParams &p, int i, Tile &t) const {
        if (i >= count) return false;
        if (MODE == GROUPED_DW) {
            const int n = tiles_m * tiles_c;
            const int flat = lo + i;
            t.e = per > 0 ? i / per : flat / n;
            const int at = per > 0 ? lo + i % per : flat % n;
            t.m0 = at % tiles_m * TM;
            t.c0 = at / tiles_m * TM;
            t.m_end = p.N;
            t.c_end = p.K;
            int end;
            group_rows(p.offsets, t.e, p.R, t.r0, end);
            t.red = end - t.r0;
            return true;
        }
        const int at = lo + i;
        const int band = at / (8 * tiles_c), in = at - band * 8 * tiles_c;
        const int height = min(8, tiles_m - band * 8);
        const int rt = band * 8 + in % height;
        t.c0 = in / height * TM;
        int a = 0, b = p.E;            // the group whose row tiles hold rt
        while (b - a > 1) {
            const int mid = (a + b) >> 1;
            if (prefix[mid] <= rt)
                a = mid;
            else
                b = mid;
        }
        t.e = a;
        int first, end;
        group_rows(p.offsets, a, p.R, first, end);
        t.m0 = first + (rt - prefix[a]) * TM;
        t.m_end = min(end, t.m0 + TM);
        t.c_end = MODE == GROUPED_FWD ? p.N : p.K;
        t.r0 = 0;
        t.red = MODE == GROUPED_FWD ? p.K : p.N;
        return true;
    }
};

template <int MODE, bool VEC>
__global__ __launch_bounds__(TILE_THREADS) void grouped_tile_kernel(GroupedParams p) {
    extern __shared__ __attribute__((aligned(16))) char tile_lds[];
    typedef TileShape<MODE> Shape;
    const int tid = threadIdx.x, lane = tid & 63;
    int *prefix = reinterpret_cast<int *>(tile_lds + 2 * Shape::STAGE);

    TileList<MODE> list;
    list.prefix = prefix;
    list.tiles_c = ((MODE == GROUPED_FWD ? p.N : p.K) + TM - 1) / TM;
    if (MODE == GROUPED_DW) {
        list.tiles_m = (p.N + TM - 1) / TM;
        const int n = list.tiles_m * list.tiles_c, x = blockIdx.x & 7;
        const bool shared = n >= 64;
        const long long part = shared ? n : (long long)n * p.E;
        list.lo = (int)(part * x / 8);
        list.count = (int)(part * (x + 1) / 8) - list.lo;
        list.per = shared ? list.count : 0;
        if (shared) list.count *= p.E;
    } else {
        // one wave sums the row tiles of the groups
        if (tid < 64) {
            int carry = 0;
            for (int e0 = 0; e0 < p.E; e0 += 64) {
                const int e = e0 + lane;
                int first = 0, end = 0;
                if (e < p.E) group_rows(p.offsets, e, p.R, first, end);
                const int tiles = (end - first + TM - 1) / TM;
                int inc = tiles;
#pragma unroll
                for (int off = 1; off < 64; off <<= 1) {
                    const int u = __shfl_up(inc, off, 64);
                    if (lane >= off) inc += u;
                }
                if (e < p.E) prefix[e] = carry + inc - tiles;
                carry += __shfl(inc, 63, 64);
            }
            if (lane == 0) prefix[p.E] = carry;
        }
        __syncthreads();
        list.tiles_m = prefix[p.E];
        const long long total = (long long)list.tiles_m * list.tiles_c;
        list.lo = (int)(total * (blockIdx.x & 7) / 8);
        list.count = (int)(total * ((blockIdx.x & 7) + 1) / 8) - list.lo;
    }
    const int first = blockIdx.x >> 3, step = gridDim.x >> 3;

    int buf = 0;
    if (tid < 256) {
        // ---- loads, splits, writes
        const bool rows_side = tid < 128;
        const int u = tid & 127;
        auto walk = [&](auto stager, int side) {
            Tile t;
            for (int i = first; list.get(p, i, t); i += step) {
                if (t.red == 0) continue;
                const int stages = (t.red + TK - 1) / TK;
                stager.start(p, t, u);
                stager.load(0);
                for (int s = 0; s < stages; s++) {
                    auto now = stager;
                    if (s + 1 < stages) stager.load(s + 1);
                    now.write(tile_lds + buf * Shape::STAGE + side * Shape::SIDE, s, u);
                    buf ^= 1;
                    stage_barrier();
                }
            }
            // the barrier behind the last stage's matrix work
            stage_barrier();
        };
        if (rows_side) {
            if constexpr (Shape::AK)
                walk(StageK<MODE, true, VEC>(), 0);
            else
                walk(StageM<MODE, true, VEC>(), 0);
        } else {
            if constexpr (Shape::BK)
                walk(StageK<MODE, false, VEC>(), 1);
            else
                walk(StageM<MODE, false, VEC>(), 1);
        }
        return;
    }
    // ---- fragments, matrix instructions, results
    const int cw = (tid >> 6) - 4, wm = cw >> 1, wn = cw & 1;
    const int frag = (lane >> 5) * PLANE + (lane & 31) * 16;
    const int a_at = frag + wm * 64 * 16, b_at = Shape::SIDE + frag + wn * 64 * 16;
    stage_barrier();
    Tile t;
    for (int i = first; list.get(p, i, t); i += step) {
        floatx16 acc[2][2][2];
#pragma unroll
        for (int q = 0; q < 2; q++)
#pragma unroll
            for (int x = 0; x < 2; x++)
#pragma unroll
                for (int y = 0; y < 2; y++)
#pragma unroll
                    for (int v = 0; v < 16; v++) acc[q][x][y][v] = 0.f;
        const int stages = (t.red + TK - 1) / TK;
        for (int s = 0; s < stages; s++) {
            const char *st = tile_lds + buf * Shape::STAGE;
#pragma unroll
            for (int o = 0; o < Shape::OPS; o++) {
                bf16x8 a[2][3], b[2][3];
#pragma unroll
                for (int q = 0; q < 3; q++)
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        a[x][q] = *reinterpret_cast<const bf16x8 *>(st + a_at + (o * 3 + q) * 2 * PLANE + x * 32 * 16);
                        b[x][q] = *reinterpret_cast<const bf16x8 *>(st + b_at + (o * 3 + q) * 2 * PLANE + x * 32 * 16);
                    }
                constexpr int PA[6] = {0, 0, 1, 1, 0, 2}, PB[6] = {0, 1, 0, 1, 2, 0};
#pragma unroll
                for (int q = 0; q < 6; q++)
#pragma unroll
                    for (int x = 0; x < 2; x++)
#pragma unroll
                        for (int y = 0; y < 2; y++)
                            acc[o > 0][x][y] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                                a[x][PA[q]], b[y][PB[q]], acc[o > 0][x][y], 0, 0, 0);
            }
            buf ^= 1;
            stage_barrier();
        }
        // register v of lane l: row 8 (v / 4) + 4 (l / 32) + v % 4, column l % 32
        if constexpr (VEC && !Shape::BK) {
            // the two column sub-tiles hold neighbouring columns
            const int c = t.c0 + row_at<false>(wn * 64 + (lane & 31));
            if (c >= t.c_end) continue;
            const size_t base = (MODE == GROUPED_DW ? (size_t)t.e * p.N * p.K : 0) + c;
#pragma unroll
            for (int x = 0; x < 2; x++) {
                float2 f[16];
                size_t at[16];
#pragma unroll
                for (int v = 0; v < 16; v++) {
                    const int pos = wm * 64 + x * 32 + 8 * (v >> 2) + 4 * (lane >> 5) + (v & 3);
                    const int m = t.m0 + row_at<Shape::AK>(pos);
                    at[v] = base + (size_t)min(m, t.m_end - 1) * p.K;
                    f[v] = p.e0 != nullptr ? *reinterpret_cast<const float2 *>(p.e0 + at[v])
                                           : make_float2(1.f, 1.f);
                }
#pragma unroll
                for (int v = 0; v < 16; v++) {
                    const int pos = wm * 64 + x * 32 + 8 * (v >> 2) + 4 * (lane >> 5) + (v & 3);
                    if (t.m0 + row_at<Shape::AK>(pos) >= t.m_end) continue;
                    *reinterpret_cast<float2 *>(p.out0 + at[v]) =
                        make_float2(acc[0][x][0][v] * f[v].x, acc[0][x][1][v] * f[v].y);
                    *reinterpret_cast<float2 *>(p.out1 + at[v]) = make_float2(
                        acc[1][x][0][v] * f[v].x * f[v].x, acc[1][x][1][v] * f[v].y * f[v].y);
                }
            }
            continue;
        }
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
            for (int y = 0; y < 2; y++) {
                const int c = t.c0 + row_at<Shape::BK>(wn * 64 + y * 32 + (lane & 31));
                if (c >= t.c_end) continue;
                float b0 = 0.f, b1 = 0.f;
                if (MODE == GROUPED_FWD && p.e0 != nullptr) {
                    b0 = p.e0[(size_t)t.e * p.N + c];
                    b1 = p.e1[(size_t)t.e * p.N + c];
                }
#pragma unroll
                for (int v = 0; v < 16; v++) {
                    const int pos = wm * 64 + x * 32 + 8 * (v >> 2) + 4 * (lane >> 5) + (v & 3);
                    const int m = t.m0 + row_at<Shape::AK>(pos);
                    if (m >= t.m_end) continue;
                    const float s0 = acc[0][x][y][v], s1 = acc[1][x][y][v];
                    if (MODE == GROUPED_FWD) {
                        store_activated(p.act, s0 + b0, s1 + b1, (size_t)m * p.N + c, p.out0, p.out1, p.out2);
                    } else {
                        const size_t at = (MODE == GROUPED_DW ? (size_t)t.e * p.N * p.K : 0) + (size_t)m * p.K + c;
                        const float f = p.e0 != nullptr ? p.e0[at] : 1.f;
                        p.out0[at] = s0 * f;
                        p.out1[at] = s1 * f * f;
                    }
                }
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
inline bool aligned16(const void *q) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0; }

template <int MODE, bool VEC>
hipError_t tile_launch(const GroupedParams &p, long long tiles, hipStream_t stream) {
    static PerDeviceOnce once;
    const int lds = TileShape<MODE>::LDS;
    hipError_t e = allow_dynamic_lds(
        once, reinterpret_cast<const void *>(&grouped_tile_kernel<MODE, VEC>), lds);
    if (e != hipSuccess) return e;
    // one workgroup per CU at most; every XCD the same number
    const long long most = num_cu() / 8 * 8, want = (tiles + 7) / 8 * 8;
    hipLaunchKernelGGL((grouped_tile_kernel<MODE, VEC>), dim3((unsigned)(want < most ? want : most)),
                       dim3(TILE_THREADS), lds, stream, p);
    return hipGetLastError();
}

template <bool VEC>
hipError_t tile_launch(GroupedMode mode, const GroupedParams &p, hipStream_t stream) {
    // row tiles over all groups: every group ends with at most one part tile
    const long long row_tiles = p.R / TM + (p.E < p.R ? p.E : p.R);
    if (mode == GROUPED_FWD) return tile_launch<GROUPED_FWD, VEC>(p, row_tiles * ceil_div(p.N, TM), stream);
    if (mode == GROUPED_DZ) return tile_launch<GROUPED_DZ, VEC>(p, row_tiles * ceil_div(p.K, TM), stream);
    return tile_launch<GROUPED_DW, VEC>(p, (long long)ceil_div(p.K, TM) * ceil_div(p.N, TM) * p.E, stream);
}

}  // namespace

hipError_t launch_grouped(GroupedMode mode, const GroupedParams &p, hipStream_t stream) {
    // 16-byte loads: every row of every operand starts on 16 bytes
    const bool vec = p.K % 4 == 0 && (mode == GROUPED_FWD || p.N % 4 == 0) && aligned16(p.x0) &&
                     aligned16(p.x1) && aligned16(p.y0) && (mode != GROUPED_FWD || aligned16(p.y1)) &&
                     (mode == GROUPED_FWD || (aligned16(p.e0) && aligned16(p.out0) && aligned16(p.out1)));
    return vec ? tile_launch<true>(mode, p, stream) : tile_launch<false>(mode, p, stream);
}

hipError_t launch_grouped_db(const GroupedParams &p, hipStream_t stream) {
    hipLaunchKernelGGL(grouped_db_kernel, dim3(ceil_div(p.N, 64), p.E), dim3(TPB), 0, stream, p);
    return hipGetLastError();
}

}  // namespace tagi
