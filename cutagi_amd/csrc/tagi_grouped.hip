// Linear layers grouped by expert: row r of expert e (offsets[e] <= r < offsets[e+1])
// meets the weights [e][N][K]. gfx950.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "tagi_activation.h"
#include "tagi_grouped.h"
#include "tagi_internal.h"

namespace tagi {

int g_grouped_rows = -1;

namespace {

constexpr int TPB = 256;
constexpr int MAX_GROUPS = 1024;

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
// fp32 arithmetic would give an infinity or NaN. The last part of a number below 2^-108 (3e-33)
// is below the normal numbers and may be lost, the middle one from 2^-117 on.
//
// A workgroup owns 128 x 128 tiles (64 x 128 where experts have few rows) of an output pair and walks them one after the other. Four
// of its waves load the operands, form the sums and squares that the variance needs, split
// them and write the pieces to LDS; the other four read fragments and issue matrix
// instructions on 64 x 64 (32 x 64) sub-tiles. Every SIMD holds one wave of each kind, so the vector
// work of the split runs under the matrix instructions without any interleaving in the code,
// and an element is split once for the two waves that read it.
// The two kinds meet at one barrier per unit, 32 reduction elements of one product (mean;
// variance, one or two), 48 matrix instructions per wave: while unit u is multiplied, its
// second half and the first half of unit u + 1 are read from LDS and unit u + 2 is written.
//
// Bound by the matrix instructions at the clock that the power limit leaves: the forward of
// 8192 rows, 8 experts of 2048 -> 4096, takes 2085 us (1.19 PFLOP/s of bf16 products, 198 TFLOP/s
// of fp32 ones, where the fp32 matrix instructions end at 157) and 1611 us with nothing but its
// matrix instructions left; the backward of 4096 -> 2048 takes 2943 us. (2815 us for the forward
// with 16-element units, half lines per load and fragments read when they were needed; 8105 us
// with fp32 products on plain tiles.)
// ---------------------------------------------------------------------------
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef float floatx16 __attribute__((ext_vector_type(16)));

// The three bf16 pieces of a and b, packed pairwise. (A two-term dot product would take a
// piece off in one instruction instead of two, but it runs on the matrix pipe and so not
// beside the matrix instructions of the other wave.)
__device__ __forceinline__ void split_pair(float a, float b, unsigned (&piece)[3]) {
#pragma unroll
    for (int s = 0; s < 3; s++) {
        piece[s] = __builtin_bit_cast(unsigned, __builtin_convertvector((floatx2){a, b}, bf16x2));
        if (s < 2) {
            a -= __uint_as_float(piece[s] << 16);
            b -= __uint_as_float(piece[s] & 0xffff0000u);
        }
    }
}

constexpr int TM = 128;             // rows (64 XM of them: forward, state backward) and columns of a tile
constexpr int TK = 32;              // reduction elements of a unit
constexpr int TILE_THREADS = 512;   // 256 that stage, 256 that multiply
// One piece of one operand of a unit: 64 bytes per row (or column) of the tile, four chunks of
// eight reduction elements, their order turned by the row so that the sixteen lanes of a
// 16-byte access (one chunk of sixteen rows) and of an 8-byte one (two whole rows) each touch
// every bank once.
constexpr int PIECE = TM * TK * 2;
constexpr int UNIT = 2 * 3 * PIECE;   // rows' pieces, then columns' pieces
constexpr int RING = 3;
constexpr int TILE_LDS = RING * UNIT + (MAX_GROUPS + 1) * 4;

__device__ __forceinline__ int chunk_at(int pos, int chunk) {
    return pos * (TK * 2) + ((chunk ^ ((pos >> 2) & 3)) << 4);
}

template <int MODE>
struct TileShape {
    static constexpr int OPS = MODE == GROUPED_FWD ? 3 : 2;         // products, operands per side
    // reduction contiguous in memory on the row / column side?
    static constexpr bool AK = MODE != GROUPED_DW, BK = MODE == GROUPED_FWD;
};

// Which row (or column) of a tile is at position pos of the LDS. Operands whose reduction
// index is the slow one are loaded four neighbouring columns at a time; these go to
// positions 32 apart, so that neighbouring lanes write neighbouring places.
template <bool KCONTIG>
__device__ __forceinline__ int row_at(int pos) {
    return KCONTIG ? pos : (pos & 31) * 4 + (pos >> 5);
}

__device__ __forceinline__ void unit_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// The same for the half that only reads: its reads may cross, because the unit they belong to
// is overwritten two barriers later, and the registers they fill are used before the next.
__device__ __forceinline__ void reader_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Operand `o` of one side from the values loaded: FWD rows (mu_a, var_a + mu_a^2, var_a), FWD
// columns (mu_w, var_w, mu_w^2), innovations (delta_mu, delta_var), DZ / DW columns (w or a,
// its square).
template <int MODE, bool ROWS>
__device__ __forceinline__ float operand(int o, float u, float v) {
    if (o == 0) return u;
    if (MODE == GROUPED_FWD) {
        if (o == 1) return ROWS ? fmaf(u, u, v) : v;
        return ROWS ? v : u * u;
    }
    return ROWS ? v : u * u;
}

// A tile of the problem: expert, first row / column, reduction range, and the rows that exist.
struct Tile {
    int e, m0, c0;      // expert, first output row, first output column
    int m_end, c_end;   // one past the last
    int r0, red;        // first element of the reduction (DW: row), their number
    int part;           // which part of a divided reduction
};

// The tiles of a workgroup: XCD x (workgroups x, x + 8, ...) takes the x-th eighth of the tile
// list, its workgroups every (workgroups of the XCD)-th tile of that.
//   FWD, DZ: row tiles over all groups, eight of them by all columns, so that the workgroups
//            of an XCD share rows and columns in its L2
//   DW: the same eighth of every expert's tiles, whatever its number of rows; an eighth of
//            all experts' tiles in order where an expert has too few to divide
// A divided reduction has all tiles once per part; the parts are whole units.
template <int MODE, int XM>
struct TileList {
    int tiles_m, tiles_c, lo, count;   // this XCD's part of the list
    int per;                           // DW: tiles of it per expert and part, 0: of all in order
    const int *prefix;                 // row tiles before every group (LDS)
    // the part-th of p.splits parts of a reduction
    static __device__ __forceinline__ void divide(const GroupedParams &p, Tile &t) {
        if (p.splits == 1) return;
        const int units = (t.red + TK - 1) / TK;
        const int lo = (int)((long long)units * t.part / p.splits) * TK;
        const int hi = (int)((long long)units * (t.part + 1) / p.splits) * TK;
        t.red = min(hi, t.red) - lo;
        t.r0 += lo;
    }
    __device__ __forceinline__ bool get(const GroupedParams &p, int i, Tile &t) const {
        if (i >= count) return false;
        if (MODE == GROUPED_DW) {
            const int n = tiles_m * tiles_c;
            const int flat = lo + i;
            const int each = per > 0 ? i / per : flat / n;
            t.e = each % p.E;
            t.part = each / p.E;
            const int at = per > 0 ? lo + i % per : flat % n;
            t.m0 = at % tiles_m * TM;
            t.c0 = at / tiles_m * TM;
            t.m_end = p.N;
            t.c_end = p.K;
            int end;
            group_rows(p.offsets, t.e, p.R, t.r0, end);
            t.red = end - t.r0;
            divide(p, t);
            return true;
        }
        t.part = (lo + i) / (tiles_m * tiles_c);
        const int at = lo + i - t.part * tiles_m * tiles_c;
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
        t.m0 = first + (rt - prefix[a]) * (64 * XM);
        t.m_end = min(end, t.m0 + 64 * XM);
        t.c_end = MODE == GROUPED_FWD ? p.N : p.K;
        t.r0 = 0;
        t.red = MODE == GROUPED_FWD ? p.K : p.N;
        divide(p, t);
        return true;
    }
};

// What the 128 threads that stage one side hold of 32 reduction elements.
struct Batch {
    float4_any v0[8], v1[8];
    int left;       // reduction elements from the first of the batch to the end
    int shift;      // columns by which the loads were moved to end with their row
    unsigned dead;  // bit i: v[i] belongs to no row and reads as zeros
};

// Four neighbouring floats at element `off` behind a uniform base, at a 32-bit byte offset
// (launch_grouped sees to the sizes) or, FAR, a 64-bit one.
template <bool FAR>
__device__ __forceinline__ float4_any load4(const float *base, unsigned off) {
    if (FAR) return *reinterpret_cast<const float4_any *>(base + off);
    return *reinterpret_cast<const float4_any *>(reinterpret_cast<const char *>(base) + off * 4u);
}
// v moved by n elements to the front, zeros behind them (0 <= n <= 4)
__device__ __forceinline__ float4_any to_front(float4_any v, int n) {
    const bool one = n & 1, two = n & 2, all = n & 4;
    v = one ? (float4_any){v[1], v[2], v[3], 0.f} : v;
    v = two ? (float4_any){v[2], v[3], 0.f, 0.f} : v;
    return all ? (float4_any){0.f, 0.f, 0.f, 0.f} : v;
}

// Side with its reduction index contiguous: thread u holds the elements 4 (u % 8) .. + 3 of
// the NR rows u / 8 + 16 i: eight lanes read a whole 128-byte line. At the end of a reduction
// that is no multiple of four the loads are moved to end with their row, and what they bring
// is moved back before the split.
template <int MODE, bool ROWS, bool FAR, int NR>
struct SideK {
    static constexpr int LOADS = NR;
    const float *q0, *q1;       // uniform
    static constexpr bool GATHER = ROWS && MODE == GROUPED_FWD;
    unsigned row[NR];           // element offset of the thread's rows
    int source[GATHER ? NR : 1]; // gather: the rows of the next tile
    bool fresh, gather;
    unsigned dead;
    int k, red, at, first_row, last_row;
    const float *f0, *f1;       // the batch that is loaded
    __device__ __forceinline__ void start(const GroupedParams &p, const Tile &t, int u) {
        k = (u & 7) * 4;
        red = t.red;
        fresh = true;
        gather = GATHER && p.rows != nullptr;
        const size_t first = gather ? 0 : ROWS ? (size_t)t.m0 : (size_t)t.e * p.N + t.c0;
        const size_t from = first * (MODE == GROUPED_FWD ? p.K : p.N) + t.r0;
        q0 = (ROWS ? p.x0 : p.y0) + from;
        q1 = (ROWS ? p.x1 : p.y1) + from;
        first_row = u >> 3;
        last_row = (ROWS ? t.m_end - t.m0 : t.c_end - t.c0) - 1;
        if constexpr (GATHER) {
            if (gather)
#pragma unroll
                for (int i = 0; i < NR; i++) source[i] = p.rows[t.m0 + min(first_row + 16 * i, last_row)];
        }
    }
    __device__ __forceinline__ void ahead(const GroupedParams &, int) {}
    // The batch at k0 is next: everything that its loads need. (They go out after start() may
    // have moved this side on to the next tile.)
    __device__ __forceinline__ void begin(const GroupedParams &p, int k0, Batch &b) {
        if (fresh) {
            fresh = false;
            dead = 0u;
#pragma unroll
            for (int i = 0; i < NR; i++) {
                int s = min(first_row + 16 * i, last_row);
                if constexpr (GATHER) {
                    if (gather) s = source[i];
                    if (gather && (unsigned)s >= (unsigned)p.T) {
                        s = 0;
                        dead |= 1u << i;
                    }
                }
                row[i] = (unsigned)s * (unsigned)(MODE == GROUPED_FWD ? p.K : p.N);
            }
        }
        b.left = red - k0;
        b.shift = 0;
        b.dead = dead;
        const bool whole = b.left >= TK;
        at = whole ? k : min(k0 + k, red - 4);
        f0 = q0 + (whole ? k0 : 0);
        f1 = q1 + (whole ? k0 : 0);
    }
    // its i-th load of array `second`
    __device__ __forceinline__ void load(Batch &b, int i, bool second) const {
        (second ? b.v1 : b.v0)[i] = load4<FAR>(second ? f1 : f0, row[i] + at);
    }
    // zeros behind the end of the reduction and in rows that are no rows
    __device__ __forceinline__ void mask(Batch &b) const {
#pragma unroll
        for (int i = 0; i < NR; i++) {
            const int over = (b.dead >> i) & 1u ? 4 : min(max(4 - (b.left - k), 0), 4);
            b.v0[i] = to_front(b.v0[i], over);
            b.v1[i] = to_front(b.v1[i], over);
        }
    }
    // Operand O of the batch to LDS. The loads of the batch after it go out between the
    // splits, the first array's under the first operand, the second's under the second: all
    // at once they would fill the memory pipe's queue and hold the splits up behind it.
    template <int O>
    __device__ __forceinline__ void write(const Batch &b, char *side, int u, Batch *next) const {
        char *to = side + chunk_at(u >> 3, (u & 7) >> 1) + (u & 1) * 8;
#pragma unroll
        for (int i = 0; i < NR; i++) {
            if (O < 2 && next != nullptr) load(*next, i, O == 1);
            const float4_any x = b.v0[i], y = b.v1[i];
            unsigned lo[3], hi[3];
            split_pair(operand<MODE, ROWS>(O, x[0], y[0]), operand<MODE, ROWS>(O, x[1], y[1]), lo);
            split_pair(operand<MODE, ROWS>(O, x[2], y[2]), operand<MODE, ROWS>(O, x[3], y[3]), hi);
#pragma unroll
            for (int s = 0; s < 3; s++)
                *reinterpret_cast<uint2 *>(to + s * PIECE + i * 16 * TK * 2) = make_uint2(lo[s], hi[s]);
        }
    }
};

// Side with its reduction index slow: thread u holds the columns 4 (u % 32) .. + 3 of the
// reduction elements 8 (u / 32) + i: 32 lanes read 512 bytes of one.
template <int MODE, bool ROWS, bool FAR>
struct SideM {
    static constexpr int LOADS = 8;
    static constexpr bool GATHER = MODE == GROUPED_DW && !ROWS;
    const float *q0, *q1;     // element (reduction 0, column 0) of the operand, uniform
    int ld, red, r0, g, col, shift;
    bool gather;
    int source[8];            // gather: the rows that the next batch reads
    unsigned row[8];          // the batch that is loaded: the thread's elements in its rows
    const float *f0, *f1;
    __device__ __forceinline__ void start(const GroupedParams &p, const Tile &t, int u) {
        g = (u >> 5) * 8;
        red = t.red;
        r0 = t.r0;
        gather = GATHER && p.rows != nullptr;
        if (ROWS) {             // DW: innovations [R][N], columns n
            ld = p.N;
            q0 = p.x0 + (size_t)t.r0 * p.N;
            q1 = p.x1 + (size_t)t.r0 * p.N;
        } else {
            ld = p.K;
            const size_t before = MODE == GROUPED_DZ ? (size_t)t.e * p.N + t.r0 : gather ? 0 : (size_t)t.r0;
            q0 = p.y0 + before * p.K;
            q1 = q0;
        }
        // (columns beyond the last are computed and not stored; they only have to exist)
        const int want = (ROWS ? t.m0 : t.c0) + (u & 31) * 4;
        col = min(want, ld - 4);
        shift = want - col;
    }
    // the row indices of the batch at k0, on their way while the batch before it is split
    __device__ __forceinline__ void ahead(const GroupedParams &p, int k0) {
        if (!GATHER || !gather) return;
#pragma unroll
        for (int i = 0; i < 8; i++) source[i] = p.rows[r0 + min(k0 + g + i, red - 1)];
    }
    __device__ __forceinline__ void begin(const GroupedParams &p, int k0, Batch &b) {
        b.left = red - k0;
        b.shift = shift;
        b.dead = 0u;
        f0 = q0 + (GATHER && gather ? 0 : (size_t)k0 * ld);
        f1 = q1 + (size_t)k0 * ld;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            int s = min(g + i, b.left - 1);
            if (GATHER && gather) {
                s = source[i];
                if ((unsigned)s >= (unsigned)p.T) {
                    s = 0;
                    b.dead |= 1u << i;
                }
            }
            row[i] = (unsigned)s * (unsigned)ld + (unsigned)col;
        }
    }
    __device__ __forceinline__ void load(Batch &b, int i, bool second) const {
        if (!second)
            b.v0[i] = load4<FAR>(f0, row[i]);
        else if (ROWS)
            b.v1[i] = load4<FAR>(f1, row[i]);
    }
    __device__ __forceinline__ void mask(Batch &b) const {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int over = i >= b.left - g || (b.dead >> i) & 1u ? 4 : min(b.shift, 4);
            b.v0[i] = to_front(b.v0[i], over);
            if (ROWS) b.v1[i] = to_front(b.v1[i], over);
        }
    }
    template <int O>
    __device__ __forceinline__ void write(const Batch &b, char *side, int u, Batch *next) const {
        char *to = side + chunk_at(u & 31, u >> 5);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (next != nullptr) {
                load(*next, 2 * j, O == 1);
                load(*next, 2 * j + 1, O == 1);
            }
            unsigned x[4][3];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                auto value = [&](int r) { return operand<MODE, ROWS>(O, b.v0[r][j], ROWS ? b.v1[r][j] : 0.f); };
                split_pair(value(2 * i), value(2 * i + 1), x[i]);
            }
#pragma unroll
            for (int s = 0; s < 3; s++)
                *reinterpret_cast<uint4 *>(to + s * PIECE + j * 32 * TK * 2) =
                    make_uint4(x[0][s], x[1][s], x[2][s], x[3][s]);
        }
    }
};

// One of the two staging halves of a workgroup.
template <int MODE, int XM, typename Side>
struct Stager {
    const GroupedParams &p;
    const TileList<MODE, XM> &list;
    char *lds;
    int next, step, u;
    Side side;
    Tile t;
    int k0;
    bool more;
    int slot;

    // moves to the next batch of the tile, or the first of the next tile that has any
    __device__ __forceinline__ void advance() {
        k0 += TK;
        if (k0 >= t.red) {
            do {
                more = list.get(p, next, t);
                next += step;
            } while (more && t.red == 0);
            k0 = 0;
            if (more) side.start(p, t, u);
        }
        if (more) side.ahead(p, k0);
    }
    template <int O>
    __device__ __forceinline__ void units(const Batch &b, Batch *after) {
        if constexpr (O < TileShape<MODE>::OPS) {
            side.template write<O>(b, lds + slot * UNIT, u, after);
            slot = slot == RING - 1 ? 0 : slot + 1;
            unit_barrier();
            units<O + 1>(b, after);
        }
    }
    // batch b to LDS, the batch after it into `after`
    __device__ __forceinline__ void put(Batch &b, Batch &after) {
        if (b.left < TK || b.dead != 0u || b.shift != 0) side.mask(b);
        if (more) {
            side.begin(p, k0, after);
            advance();
            units<0>(b, &after);
        } else {
            after.left = 0;
            units<0>(b, nullptr);
        }
    }
    __device__ __forceinline__ void run() {
        Batch a, b;
        more = true;
        slot = 0;
        t.red = 0;
        k0 = 0;
        advance();
        if (more) {
            side.begin(p, k0, a);
            advance();
#pragma unroll
            for (int i = 0; i < Side::LOADS; i++) {
                side.load(a, i, false);
                side.load(a, i, true);
            }
            while (true) {
                put(a, b);
                if (b.left == 0) break;
                put(b, a);
                if (a.left == 0) break;
            }
        }
        // the two barriers by which the multiplying half is behind
        unit_barrier();
        unit_barrier();
    }
};

// The functions below take four columns to a thread; the last four of a row start at its end less
// four, so that some columns are taken twice, with the same result.
__device__ __forceinline__ void add4(float4_any &sum, const float *p) {
    sum += *reinterpret_cast<const float4_any *>(p);
}

// Bias innovations of one expert's columns, 2^db_log (up to eight) groups of four of them to a
// workgroup: the other bits of the thread index are rows, four of them in flight each. The
// row threads of a wave are joined by lane exchanges, the waves in their order. Groups of a
// workgroup 4 / 8 / 16 / 32, with the weight backward of eight inputs before it: 8192 rows, 8
// experts of 2048 outputs 140 / 120 / 122 / 133 us, of 512 50 / 47 / 54 / 70.
constexpr int DB_GROUPS = 8;

template <int WAVES>
__device__ __forceinline__ void bias_sums(const GroupedParams &p, int block, float (*s)[WAVES][DB_GROUPS * 4]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, cw = 1 << p.db_log;
    const int blocks = ((p.N + 3) / 4 + cw - 1) >> p.db_log, e = block / blocks;
    const int c0 = (block - e * blocks) * cw * 4;
    int first, end;
    group_rows(p.offsets, e, p.R, first, end);
    float4_any m[4], v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) m[i] = v[i] = (float4_any){0.f, 0.f, 0.f, 0.f};
    const int step = (WAVES * 64) >> p.db_log;
    const size_t col = min(c0 + 4 * ((int)threadIdx.x & (cw - 1)), p.N - 4);
    const float *x = p.x0 + col, *y = p.x1 + col;
    long long r = first + (threadIdx.x >> p.db_log);
    for (; r + 3 * step < end; r += 4 * step)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            add4(m[i], x + (r + i * step) * p.N);
            add4(v[i], y + (r + i * step) * p.N);
        }
    for (; r < end; r += step) {
        add4(m[0], x + r * p.N);
        add4(v[0], y + r * p.N);
    }
    m[0] = (m[0] + m[1]) + (m[2] + m[3]);
    v[0] = (v[0] + v[1]) + (v[2] + v[3]);
#pragma unroll
    for (int c = 0; c < 4; c++) {
        float sm = m[0][c], sv = v[0][c];
        for (int off = 32; off >= cw; off >>= 1) {
            sm += __shfl_xor(sm, off, 64);
            sv += __shfl_xor(sv, off, 64);
        }
        if (lane < cw) {
            s[0][wave][4 * lane + c] = sm;
            s[1][wave][4 * lane + c] = sv;
        }
    }
    __syncthreads();
    const int t = threadIdx.x, want = c0 + (t & ~3);
    if (t >= 4 * cw || want >= p.N) return;
    float sm = 0.f, sv = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; w++) {
        sm += s[0][w][t];
        sv += s[1][w][t];
    }
    const size_t at = (size_t)e * p.N + min(want, p.N - 4) + (t & 3);
    const float vb = p.e1[at];
    p.db0[at] = vb * sm;
    p.db1[at] = vb * vb * sv;
}

template <int MODE, int XM, bool FAR>
__global__ __launch_bounds__(TILE_THREADS) void grouped_tile_kernel(GroupedParams p) {
    extern __shared__ __attribute__((aligned(16))) char tile_lds[];
    typedef TileShape<MODE> Shape;
    const int tid = threadIdx.x, lane = tid & 63;
    if (MODE == GROUPED_DW && (int)blockIdx.x >= p.tile_wgs) {
        bias_sums<TILE_THREADS / 64>(p, blockIdx.x - p.tile_wgs,
                                     reinterpret_cast<float(*)[TILE_THREADS / 64][DB_GROUPS * 4]>(tile_lds));
        return;
    }
    int *prefix = reinterpret_cast<int *>(tile_lds + RING * UNIT);

    TileList<MODE, XM> list;
    list.prefix = prefix;
    list.tiles_c = ((MODE == GROUPED_FWD ? p.N : p.K) + TM - 1) / TM;
    if (MODE == GROUPED_DW) {
        list.tiles_m = (p.N + TM - 1) / TM;
        const int n = list.tiles_m * list.tiles_c, x = blockIdx.x & 7;
        const bool shared = n >= 64;
        const long long part = shared ? n : (long long)n * p.E * p.splits;
        list.lo = (int)(part * x / 8);
        list.count = (int)(part * (x + 1) / 8) - list.lo;
        list.per = shared ? list.count : 0;
        if (shared) list.count *= p.E * p.splits;
    } else {
        // one wave sums the row tiles of the groups
        if (tid < 64) {
            int carry = 0;
            for (int e0 = 0; e0 < p.E; e0 += 64) {
                const int e = e0 + lane;
                int first = 0, end = 0;
                if (e < p.E) group_rows(p.offsets, e, p.R, first, end);
                const int tiles = (end - first + 64 * XM - 1) / (64 * XM);
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
        const long long total = (long long)list.tiles_m * list.tiles_c * p.splits;
        list.lo = (int)(total * (blockIdx.x & 7) / 8);
        list.count = (int)(total * ((blockIdx.x & 7) + 1) / 8) - list.lo;
    }
    const int first = blockIdx.x >> 3, step = p.tile_wgs >> 3;

    if (tid < 256) {
        // ---- loads, splits, writes
        const int u = tid & 127;
        if (tid < 128) {
            typedef std::conditional_t<Shape::AK, SideK<MODE, true, FAR, 4 * XM>, SideM<MODE, true, FAR>> Side;
            Stager<MODE, XM, Side> s{p, list, tile_lds, first, step, u};
            s.run();
        } else {
            typedef std::conditional_t<Shape::BK, SideK<MODE, false, FAR, 8>, SideM<MODE, false, FAR>> Side;
            Stager<MODE, XM, Side> s{p, list, tile_lds + 3 * PIECE, first, step, u};
            s.run();
        }
        return;
    }
    // ---- fragments, matrix instructions, results
    const int cw = (tid >> 6) - 4, wm = cw >> 1, wn = cw & 1;
    const char *a_base = tile_lds + wm * 32 * XM * TK * 2;
    const char *b_base = tile_lds + 3 * PIECE + wn * 64 * TK * 2;
    const int frag[2] = {chunk_at(lane & 31, lane >> 5), chunk_at(lane & 31, 2 + (lane >> 5))};
    // pieces of the half unit that is multiplied: [piece][sub-tile]
    bf16x8 a[3][XM], b[3][2];
    auto fetch = [&](auto &f, const char *base, int slot, int half, int piece) {
#pragma unroll
        for (int x = 0; x < (int)(sizeof(f) / sizeof(f[0])); x++)
            f[x] = *reinterpret_cast<const bf16x8 *>(base + slot * UNIT + frag[half] + piece * PIECE + x * 32 * TK * 2);
    };
    reader_barrier();
#pragma unroll
    for (int q = 0; q < 3; q++) {
        fetch(a[q], a_base, 0, 0, q);
        fetch(b[q], b_base, 0, 0, q);
    }
    reader_barrier();
    int slot = 0;
    Tile t;
    for (int i = first; list.get(p, i, t); i += step) {
        floatx16 acc[2][XM][2];
#pragma unroll
        for (int q = 0; q < 2; q++)
#pragma unroll
            for (int x = 0; x < XM; x++)
#pragma unroll
                for (int y = 0; y < 2; y++)
#pragma unroll
                    for (int v = 0; v < 16; v++) acc[q][x][y][v] = 0.f;
        for (int k0 = 0; k0 < t.red; k0 += TK) {
#pragma unroll
            for (int o = 0; o < Shape::OPS; o++) {
                auto mul = [&](const bf16x8(&x)[XM], const bf16x8(&y)[2]) {
#pragma unroll
                    for (int i = 0; i < XM; i++)
#pragma unroll
                        for (int j = 0; j < 2; j++)
                            acc[o > 0][i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                                x[i], y[j], acc[o > 0][i][j], 0, 0, 0);
                };
                const int after = slot == RING - 1 ? 0 : slot + 1;
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    // the small products first; a piece is read anew, for the next half unit, as
                    // soon as its last product is issued (the high ones are needed to the end)
                    const int from = half == 0 ? slot : after, other = 1 - half;
                    bf16x8 ah[XM], bh[2];
                    fetch(ah, a_base, from, other, 0);
                    fetch(bh, b_base, from, other, 0);
                    mul(a[2], b[0]);
                    __builtin_amdgcn_sched_barrier(0);
                    fetch(a[2], a_base, from, other, 2);
                    mul(a[0], b[2]);
                    __builtin_amdgcn_sched_barrier(0);
                    fetch(b[2], b_base, from, other, 2);
                    mul(a[1], b[1]);
                    mul(a[1], b[0]);
                    __builtin_amdgcn_sched_barrier(0);
                    fetch(a[1], a_base, from, other, 1);
                    mul(a[0], b[1]);
                    __builtin_amdgcn_sched_barrier(0);
                    fetch(b[1], b_base, from, other, 1);
                    mul(a[0], b[0]);
#pragma unroll
                    for (int x = 0; x < XM; x++) a[0][x] = ah[x];
#pragma unroll
                    for (int y = 0; y < 2; y++) b[0][y] = bh[y];
                }
                slot = after;
                reader_barrier();
            }
        }
        float *out0 = p.out0 + t.part * p.part, *out1 = p.out1 + t.part * p.part;
        // register v of lane l: row 8 (v / 4) + 4 (l / 32) + v % 4, column l % 32
        if constexpr (!Shape::BK) {
            // The two column sub-tiles hold neighbouring columns; four rows at a time. All sums are
            // scaled before any is stored, with three groups of factors on their way: a load
            // behind stores would be waited for together with them (256 rows, 8 experts of
            // 2048 -> 2048, weight backward, loads and stores in turn / apart: 157 / 112 us).
            const int c = t.c0 + row_at<false>(wn * 64 + (lane & 31));
            if (c >= t.c_end) continue;
            const bool both = c + 1 < t.c_end;
            const size_t base = (MODE == GROUPED_DW ? (size_t)t.e * p.N * p.K : 0) + c;
            constexpr int GROUPS = XM * 4;
            auto row = [&](int g, int v, int half) {
                return t.m0 + row_at<Shape::AK>((wm * XM + g / 4) * 32 + 8 * (g % 4) + 4 * half + v);
            };
            int half = lane >> 5;
            if (p.e0 != nullptr) {
                constexpr int AHEAD = 3;
                float2_any f[AHEAD][4];
                auto load = [&](int g) {
#pragma unroll
                    for (int v = 0; v < 4; v++)   // (the last column alone: with the one before it)
                        f[g % AHEAD][v] = *reinterpret_cast<const float2_any *>(
                            p.e0 + base - (both ? 0 : 1) + (size_t)min(row(g, v, half), t.m_end - 1) * p.K);
                };
#pragma unroll
                for (int g = 0; g < AHEAD; g++) load(g);
#pragma unroll
                for (int g = 0; g < GROUPS; g++) {
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int v = 0; v < 4; v++) {
                        const float2_any w = f[g % AHEAD][v];
                        const float w0 = both ? w[0] : w[1], w1 = w[1];
                        const int x = g / 4, i = 4 * (g % 4) + v;
                        acc[0][x][0][i] *= w0;
                        acc[0][x][1][i] *= w1;
                        acc[1][x][0][i] *= w0 * w0;
                        acc[1][x][1][i] *= w1 * w1;
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    if (g + AHEAD < GROUPS) load(g + AHEAD);
                }
            }
            asm volatile("" : "+v"(half));   // (the addresses are not worth keeping until here)
#pragma unroll
            for (int g = 0; g < GROUPS; g++) {
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int v = 0; v < 4; v++) {
                    const int m = row(g, v, half), x = g / 4, i = 4 * (g % 4) + v;
                    if (m >= t.m_end) continue;
                    const size_t at = base + (size_t)m * p.K;
                    if (both) {
                        *reinterpret_cast<float2_any *>(out0 + at) = (float2_any){acc[0][x][0][i], acc[0][x][1][i]};
                        *reinterpret_cast<float2_any *>(out1 + at) = (float2_any){acc[1][x][0][i], acc[1][x][1][i]};
                    } else {
                        out0[at] = acc[0][x][0][i];
                        out1[at] = acc[1][x][0][i];
                    }
                }
            }
        } else {
            float b0[2] = {0.f, 0.f}, b1[2] = {0.f, 0.f};
            const int c0 = t.c0 + wn * 64 + (lane & 31);
            if (p.e0 != nullptr)   // (ahead of all stores, as above)
#pragma unroll
                for (int y = 0; y < 2; y++) {
                    const size_t at = (size_t)t.e * p.N + min(c0 + y * 32, p.N - 1);
                    b0[y] = p.e0[at];
                    b1[y] = p.e1[at];
                }
#pragma unroll
            for (int x = 0; x < XM; x++)
#pragma unroll
                for (int y = 0; y < 2; y++) {
                    const int c = c0 + y * 32;
                    if (c >= t.c_end) continue;
#pragma unroll
                    for (int v = 0; v < 16; v++) {
                        const int m = t.m0 + (wm * XM + x) * 32 + 8 * (v >> 2) + 4 * (lane >> 5) + (v & 3);
                        if (m >= t.m_end) continue;
                        store_activated(p.act, acc[0][x][y][v] + b0[y], acc[1][x][y][v] + b1[y],
                                        (size_t)m * p.N + c, out0, out1, p.out2);
                    }
                }
        }
    }
}

// The parts of a divided reduction, in order, and what the tile kernel would have done with
// their sums (p.x0, p.x1: the parts' outputs).
constexpr int JOIN_ROWS = 8;
template <int MODE>
__global__ __launch_bounds__(TPB) void grouped_join_kernel(GroupedParams p) {
    size_t at, bias = 0;
    if (MODE == GROUPED_DW) {
        const size_t i = 4 * ((size_t)blockIdx.x * TPB + threadIdx.x);
        if (i >= p.part) return;
        at = min(i, p.part - 4);
    } else {
        // blockIdx.x: up to eight rows of one expert, the threads share their groups of columns
        int r0, end;
        const int e = find_rows(p.offsets, p.E, p.R, JOIN_ROWS, blockIdx.x, r0, end);
        if (e < 0) return;
        const int cols = MODE == GROUPED_FWD ? p.N : p.K, groups = (cols + 3) / 4;
        const int i = blockIdx.y * TPB + threadIdx.x, r = r0 + i / groups;
        if (i / groups >= JOIN_ROWS || r >= end) return;
        const int c = min(4 * (i % groups), cols - 4);
        at = (size_t)r * cols + c;
        bias = (size_t)e * cols + c;
    }
    float4_any m = {0.f, 0.f, 0.f, 0.f}, v = {0.f, 0.f, 0.f, 0.f}, f = {1.f, 1.f, 1.f, 1.f};
    if (MODE != GROUPED_FWD && p.e0 != nullptr) f = *reinterpret_cast<const float4_any *>(p.e0 + at);
#pragma unroll 4
    for (int s = 0; s < p.splits; s++) {
        add4(m, p.x0 + s * p.part + at);
        add4(v, p.x1 + s * p.part + at);
    }
    if (MODE == GROUPED_FWD) {
        if (p.e0 != nullptr) {
            add4(m, p.e0 + bias);
            add4(v, p.e1 + bias);
        }
#pragma unroll
        for (int c = 0; c < 4; c++) store_activated(p.act, m[c], v[c], at + c, p.out0, p.out1, p.out2);
        return;
    }
    *reinterpret_cast<float4_any *>(p.out0 + at) = m * f;
    *reinterpret_cast<float4_any *>(p.out1 + at) = v * f * f;
}

constexpr int DB_WAVES = 16;
__global__ __launch_bounds__(DB_WAVES * 64) void grouped_db_kernel(GroupedParams p) {
    __shared__ float s[2][DB_WAVES][DB_GROUPS * 4];
    bias_sums<DB_WAVES>(p, blockIdx.x, s);
}

inline int ceil_div(int a, int b) { return (a + b - 1) / b; }

template <int MODE, int XM, bool FAR>
hipError_t tile_launch(const GroupedParams &p, unsigned wgs, hipStream_t stream) {
    static PerDeviceOnce once;
    hipError_t e = allow_dynamic_lds(
        once, reinterpret_cast<const void *>(&grouped_tile_kernel<MODE, XM, FAR>), TILE_LDS);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((grouped_tile_kernel<MODE, XM, FAR>), dim3(wgs), dim3(TILE_THREADS), TILE_LDS, stream, p);
    return hipGetLastError();
}

// Byte offsets from a tile's first row fit 32 bits (K, N <= 2^22), those of gathered rows while
// the activations have fewer than 2^30 elements.
bool far_offsets(const GroupedParams &p) {
    return (p.rows != nullptr && (long long)p.T * p.K >= (1LL << 30)) || p.K > (1 << 22) || p.N > (1 << 22);
}

// How a call runs on the tiles: their height, parts of the reduction, and the time in us that
// this is expected to take (fitted to the measurements here).
//   Height: with up to 64 rows per expert a tile of 128 is half empty, with more it reads the
//   weights half as often. 64 / 128 rows: 256 rows, 8 experts of 2048 -> 4096: forward 189 /
//   255, state backward 123 / 170 us; 512 rows: 313 / 254, 206 / 177.
//   Parts: few tiles of long reductions leave most of the chip idle. In parts / in one piece:
//   8000 rows of 4096 -> 128: forward 158 / 367 us; 6826 rows, 2 experts of 529 -> 20: weight
//   backward 42 / 350 us.
// Groups of up to `rows` rows: of experts that are 30% smaller, average and 30% larger.
double row_groups(int R, int used, int rows) {
    const double each = (double)R / used / rows;
    return used * (std::ceil(0.7 * each) + std::ceil(each) + std::ceil(1.3 * each)) / 3;
}

struct TilePlan {
    int xm, splits;    // 64 xm rows to a tile
    long long tiles;   // at most
    double us;
};
constexpr int MAX_SPLITS = 16;

TilePlan plan_tiles(GroupedMode mode, const GroupedParams &p) {
    const int used = p.E < p.R ? p.E : p.R;
    const int cols = mode == GROUPED_FWD ? p.N : p.K;
    const int red = mode == GROUPED_FWD ? p.K : mode == GROUPED_DZ ? p.N : p.R / used;
    const int units = ceil_div(red, TK);
    const double out = mode == GROUPED_DW ? (double)p.E * p.N * p.K : (double)p.R * cols;
    const double room = (double)grouped_scratch_floats(p.K, p.N, p.E, p.R);
    TilePlan best = {2, 1, 0, 1e30};
    const bool both = mode != GROUPED_DW && !far_offsets(p);
    for (int xm = both ? 1 : 2; xm <= 2; xm++) {
        const long long rows = (long long)row_groups(p.R, used, 64 * xm), most = p.R / (64 * xm) + used;
        const long long blocks = ceil_div(cols, TM);
        const long long tiles = mode == GROUPED_DW ? (long long)ceil_div(p.K, TM) * ceil_div(p.N, TM) * p.E : rows * blocks;
        const double unit_us = mode == GROUPED_FWD ? (xm == 1 ? 2.4 : 3.2) : (xm == 1 ? 1.4 : 2.0);
        // Four units to a part at least; the parts are written and read once more, and have to
        // run at once (with some room, where the tiles depend on the experts' rows).
        for (int s = 1; s <= MAX_SPLITS; s++) {
            const long long wgs = tiles * s + (mode == GROUPED_DW || used == 1 ? 0 : tiles * s / 4);
            if (s > 1 && (wgs > num_cu() || units / s < 4 || 2 * out * s > room)) break;
            const double us = s == 1 ? 12 + unit_us * ((tiles + num_cu() - 1) / num_cu()) * units
                                     : 22 + unit_us * ceil_div(units, s) + 16 * out * s / 4e6;
            if (us < best.us) best = {xm, s, s * (mode == GROUPED_DW ? tiles : most * blocks), us};
        }
    }
    return best;
}

// Which kernels a call goes to. Up to sixteen rows per expert on average the weights are what
// takes the time, and the kernels for few rows read them once (64 rows, 16 experts of 2048 ->
// 4096: 180 against 497 us). Beyond that those also win where the tiles are too few for the
// chip, because their groups of 32 rows by 16 (forward) or 64 (state backward) outputs are
// many more, and where the tiles would be mostly empty. Measured, few rows / tiles, and the
// two formulas were fitted to these (us):
//   forward         777 rows,  6 experts,  301 ->  415   15 /  33
//                   192        8          2048 -> 4096  183 / 190
//                   256        8          2048 -> 4096  251 / 189
//                   512        8          2048 -> 4096  415 / 254
//                   512        8          1024 -> 1024   60 /  54
//                   256        4          2048 ->  512   48 /  34
//                  2048        8           512 ->  512   58 /  47
//                  1024        8          2048 -> 2048  383 / 206
//                  8000        1          4096 ->  128  399 / 145
//   state backward  777        6           301 ->  415   15 /  34
//                   192        8          2048 -> 4096   83 / 117
//                   256        8          2048 -> 4096  156 / 123
//                   512        8          2048 -> 4096  249 / 172
//                  2048        8           512 ->  512   43 /  32
//                  1024        8          2048 -> 2048  198 / 136
//                  6826        2           529 ->   20   46 /  24
// The weight backward has as many tiles as the weights: few rows only, the fewer where the
// weights are many. 8 / 12 / 16 rows per expert, few rows / tiles: 8 experts of 2048 -> 2048
// 104 / 103, 122 / 104, 139 / 105 us; 4 of 1024 -> 1024 16.5 / 22, 17.5 / 22, 20 / 22 us (with
// the launch of the bias innovations, which the kernel for few rows does itself).
bool streams(GroupedMode mode, const GroupedParams &p) {
    // (their grids: up to 1024 threads for sixteen outputs of every group of rows)
    const long long used = p.E < p.R ? p.E : p.R;
    const long long cols = mode == GROUPED_FWD ? p.N : p.K;
    if ((cols + 15) / 16 * (p.R / 16 + used) >= 1LL << 22) return false;
    if (mode == GROUPED_DW)
        return p.R <= 8LL * p.E || (p.R <= 16LL * p.E && (double)p.E * p.N * p.K <= 1 << 23);
    if (p.R <= 16LL * p.E) return true;
    const double groups = row_groups(p.R, (int)used, 32);
    const double rows_us = mode == GROUPED_FWD ? 8 + 2.4e-6 * groups * p.N * p.K
                                               : 8 + groups * (1.3e-6 * p.N * p.K + 0.02 * ceil_div(p.K, 64));
    return rows_us < plan_tiles(mode, p).us;
}

}  // namespace

size_t grouped_scratch_floats(int K, int N, int E, int R) {
    // the few-rows kernels need none
    if (K < 4 || N < 4 || (g_grouped_rows < 0 ? (long long)R <= 16LL * E : g_grouped_rows != 0)) return 0;
    // parts of two outputs: no more parts of tiles than CUs, MAX_SPLITS parts
    const double outputs = std::max((double)R * std::max(K, N), (double)E * K * N);
    return (size_t)(2 * std::min((double)num_cu() * TM * TM, MAX_SPLITS * outputs));
}

hipError_t launch_grouped(GroupedMode mode, const GroupedParams &params, hipStream_t stream) {
    GroupedParams p = params;
    // 16-byte loads are moved to stay inside their row, so a row holds four elements at least
    const bool vec = p.K >= 4 && p.N >= 4;
    if (!vec || (g_grouped_rows >= 0 ? g_grouped_rows != 0 : streams(mode, p)))
        return launch_grouped_rows(mode, p, vec, stream);
    const TilePlan plan = plan_tiles(mode, p);
    const int cols = mode == GROUPED_FWD ? p.N : p.K;
    p.splits = plan.splits;
    p.part = 0;
    GroupedParams join = p;
    if (p.splits > 1) {
        join.part = p.part = mode == GROUPED_DW ? (size_t)p.E * p.N * p.K : (size_t)p.R * cols;
        join.x0 = p.out0 = p.scratch;
        join.x1 = p.out1 = p.scratch + p.splits * p.part;
        p.e0 = nullptr;
        p.act = ACT_NONE;
    }
    const bool far = far_offsets(p), low = plan.xm == 1;
    // one workgroup per CU at most; every XCD the same number
    p.tile_wgs = (int)std::min<long long>(num_cu() / 8 * 8, (plan.tiles + 7) / 8 * 8);
    // The bias innovations go along where there are CUs left for all of them, and get a launch
    // of their own, in larger workgroups, where not (apart / along, weight backward of 777 rows,
    // 6 experts of 301 -> 415: 26 / 22 us, of 6826 rows, 2 experts of 529 -> 20: 41 / 31 us).
    unsigned wgs = p.tile_wgs, db_wgs = 0;
    if (mode == GROUPED_DW && p.db0 != nullptr) {
        while ((1 << p.db_log) < DB_GROUPS && (4 << p.db_log) < p.N) p.db_log++;
        db_wgs = (unsigned)ceil_div(ceil_div(p.N, 4), 1 << p.db_log) * p.E;
        if (wgs + db_wgs <= (unsigned)num_cu()) {
            wgs += db_wgs;
            db_wgs = 0;
        }
    }
    hipError_t e;
    if (mode == GROUPED_FWD)
        e = far   ? tile_launch<GROUPED_FWD, 2, true>(p, wgs, stream)
            : low ? tile_launch<GROUPED_FWD, 1, false>(p, wgs, stream)
                  : tile_launch<GROUPED_FWD, 2, false>(p, wgs, stream);
    else if (mode == GROUPED_DZ)
        e = far   ? tile_launch<GROUPED_DZ, 2, true>(p, wgs, stream)
            : low ? tile_launch<GROUPED_DZ, 1, false>(p, wgs, stream)
                  : tile_launch<GROUPED_DZ, 2, false>(p, wgs, stream);
    else
        e = far ? tile_launch<GROUPED_DW, 2, true>(p, wgs, stream)
                : tile_launch<GROUPED_DW, 2, false>(p, wgs, stream);
    if (e != hipSuccess) return e;
    if (p.splits > 1) {
        const dim3 grid(p.R / JOIN_ROWS + (p.E < p.R ? p.E : p.R), ceil_div(JOIN_ROWS * ((cols + 3) / 4), TPB));
        const dim3 flat((unsigned)((join.part / 4 + TPB) / TPB));
        if (mode == GROUPED_FWD)
            hipLaunchKernelGGL(grouped_join_kernel<GROUPED_FWD>, grid, dim3(TPB), 0, stream, join);
        else if (mode == GROUPED_DZ)
            hipLaunchKernelGGL(grouped_join_kernel<GROUPED_DZ>, grid, dim3(TPB), 0, stream, join);
        else
            hipLaunchKernelGGL(grouped_join_kernel<GROUPED_DW>, flat, dim3(TPB), 0, stream, join);
        e = hipGetLastError();
    }
    if (e != hipSuccess || db_wgs == 0) return e;
    hipLaunchKernelGGL(grouped_db_kernel, dim3(db_wgs), dim3(DB_WAVES * 64), 0, stream, p);
    return hipGetLastError();
}

}  // namespace tagi
