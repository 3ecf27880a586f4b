// The router of a mixture of experts and what joins its experts' outputs, for Gaussian
// activations, gfx950: choice of the experts and gates of every token, the plan that
// orders rows by expert, the gated sum and its backward pass.
#include "tagi_internal.h"
#include "tagi_stream.h"

namespace tagi {
namespace {

constexpr int TPB = 256;

// ---------------------------------------------------------------------------
// Choice. G = 2^g_log lanes hold the scores of one token, lane i the experts i, i + G, ... (NS
// of them; NS > 1 only with G = 64); top_k rounds of a maximum over the group, each of which
// takes its winner out: the lowest index among the equals, which a ballot finds. A score of
// -inf or NaN has the key 0 and is never chosen.
// The gates are the softmax of the chosen means:
//   g_j = e_j / S, e_j = exp(s_j - s_0) (s_0 is the largest), S = sum e
//   dg_j/ds_j = g_j (S - e_j) / S, with S - e_j summed from the other weights, so that a
//   gate next to one keeps its slope
// Lane j of the token keeps choice j (top_k <= 64, and <= the lanes where those are fewer).
// A round is a chain of dependent instructions and bound by their latency: the maximum goes
// through lane permutations inside the vector unit (16384 tokens, 64 experts, 4 choices, whole
// call: 129 us with the ones through LDS and 128 tokens per workgroup, 24 us with these and 32,
// of which this kernel takes 15.4, the scan 6.1 and the rows 4.1 when each is timed by itself). 32
// tokens of 16 experts go through one launch: 3.9 us.
// ---------------------------------------------------------------------------
constexpr int ROUTE_TOKENS = 32;   // tokens of a workgroup of the plan, a bit each

__device__ __forceinline__ unsigned order_bits(float s) {
    if (!(s > -INFINITY)) return 0u;
    const unsigned u = __float_as_uint(s + 0.f);   // -0 ties with 0
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float from_order_bits(unsigned k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

template <int CTRL>
__device__ __forceinline__ unsigned max_with(unsigned v) {
    return max(v, (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xF, 0xF, false));
}
// Maximum over the lane's group of 2^g_log lanes (g_log is the same for the launch).
__device__ __forceinline__ unsigned group_max(unsigned v, int g_log) {
    if (g_log >= 1) v = max_with<0xB1>(v);     // quad_perm 1 0 3 2
    if (g_log >= 2) v = max_with<0x4E>(v);     // quad_perm 2 3 0 1
    if (g_log >= 3) v = max_with<0x141>(v);    // row_half_mirror
    if (g_log >= 4) v = max_with<0x140>(v);    // row_mirror
    if (g_log == 5) v = max(v, (unsigned)__shfl_xor((int)v, 16, 64));
    if (g_log == 6) {
        const unsigned a = __builtin_amdgcn_readlane(v, 0), b = __builtin_amdgcn_readlane(v, 16);
        const unsigned c = __builtin_amdgcn_readlane(v, 32), d = __builtin_amdgcn_readlane(v, 48);
        v = max(max(a, b), max(c, d));
    }
    return v;
}

struct RouteOut {
    int *expert;              // [T][k]
    float *mu_g, *var_g, *jcb_g;
    int *offsets;             // [E + 1]
    int *token, *slot;        // [T k], [T][k]
};

// Chooses for the tokens [t0, t1) of a workgroup; every chosen (token, expert) is set in
// `mask` (LDS, [E], cleared by the caller).
template <int NS>
__device__ __forceinline__ void choose(const float *__restrict__ mu_s,
                                       const float *__restrict__ var_s, int E, int k, int t0,
                                       int t1, int g_log, const RouteOut &o, unsigned *mask) {
    const int G = 1 << g_log, lane = threadIdx.x & 63, gl = lane & (G - 1);
    const int sub = threadIdx.x >> g_log, subs = TPB >> g_log;
    const unsigned long long group = (g_log == 6 ? ~0ull : (1ull << G) - 1) << (lane - gl);
    for (int tb = t0; tb < t1; tb += subs) {
        const int t = tb + sub;
        const bool live = t < t1;   // (the exchanges below need every lane)
        unsigned key[NS];
#pragma unroll
        for (int i = 0; i < NS; i++) {
            const int e = (i << g_log) + gl;
            key[i] = live && e < E ? order_bits(mu_s[(size_t)t * E + e]) : 0u;
        }
        float top = 0.f, w = 0.f, others = 0.f;
        int chosen = -1;
        for (int j = 0; j < k; j++) {
            unsigned best = key[0];
#pragma unroll
            for (int i = 1; i < NS; i++) best = max(best, key[i]);
            best = group_max(best, g_log);
            // the winner: the first register, then the first lane that holds the maximum
            int at = -1;
#pragma unroll
            for (int i = 0; i < NS; i++) {
                const unsigned long long holds = __ballot(key[i] == best) & group;
                if (at < 0 && holds != 0ull) at = (i << g_log) + (__ffsll(holds) - 1 - (lane - gl));
            }
            if (best != 0u) {
                const float sc = from_order_bits(best);
                if (j == 0) top = sc;
                const float e = sc == top ? 1.f : expf(sc - top);   // (inf ties with inf)
                if (j == gl) {
                    w = e;
                    chosen = at;
                } else {
                    others += e;
                }
#pragma unroll
                for (int i = 0; i < NS; i++)
                    if ((i << g_log) + gl == at) key[i] = 0u;
            }
        }
        if (!live || gl >= k) continue;
        float g = 0.f, jc = 0.f, vg = 0.f;
        if (chosen >= 0) {
            const float sum = w + others;
            g = w / sum;
            jc = g * (others / sum);
            vg = jc * jc * var_s[(size_t)t * E + chosen];
            atomicOr(&mask[chosen], 1u << (t - t0));
        }
        const size_t c = (size_t)t * k + gl;
        o.expert[c] = chosen;
        o.mu_g[c] = g;
        o.var_g[c] = vg;
        o.jcb_g[c] = jc;
    }
}

// Exclusive prefix of v over the workgroup's threads; *total: the sum.
__device__ __forceinline__ int block_scan(int v, int *s, int *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int inc = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int u = __shfl_up(inc, off, 64);
        if (lane >= off) inc += u;
    }
    if (lane == 63) s[wave] = inc;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < TPB / 64; w++) {
        if (w < wave) before += s[w];
        all += s[w];
    }
    __syncthreads();
    *total = all;
    return before + inc - v;
}

// Offsets of the experts from their row counts. Thread x owns the experts x * per ... of
// consecutive per = ceil(E / TPB); count(e) gives the total, first(e) the rows of earlier
// workgroups; base[e] (LDS) becomes the first row of this workgroup's part of expert e.
template <typename Count, typename First>
__device__ __forceinline__ int expert_bases(int E, Count count, First first, int *s, int *base,
                                            int *offsets_out) {
    const int per = (E + TPB - 1) / TPB;
    const int e0 = min(E, (int)threadIdx.x * per), e1 = min(E, e0 + per);
    int mine = 0;
    for (int e = e0; e < e1; e++) mine += count(e);
    int total = 0;
    int at = block_scan(mine, s, &total);
    for (int e = e0; e < e1; e++) {
        if (offsets_out != nullptr) offsets_out[e] = at;
        base[e] = at + first(e);
        at += count(e);
    }
    if (offsets_out != nullptr && threadIdx.x == 0) offsets_out[E] = total;
    __syncthreads();
    return total;
}

// Rows of the choices of the tokens [t0, t1): base[e] + the number of earlier tokens of the
// workgroup with the same expert.
__device__ __forceinline__ void place(int k, int t0, int t1, const RouteOut &o,
                                      const unsigned *mask, const int *base) {
    for (int c = t0 * k + threadIdx.x; c < t1 * k; c += TPB) {
        const int e = o.expert[c], t = c / k;
        int row = -1;
        if (e >= 0) {
            row = base[e] + __popc(mask[e] & ((1u << (t - t0)) - 1u));
            o.token[row] = t;
        }
        o.slot[c] = row;
    }
}

// LDS: mask [E], base [E]
extern __shared__ unsigned route_lds[];

// Up to ROUTE_TOKENS tokens: everything in one workgroup.
template <int NS>
__global__ __launch_bounds__(TPB) void route_one_kernel(const float *__restrict__ mu_s,
                                                        const float *__restrict__ var_s, int T,
                                                        int E, int k, int g_log, RouteOut o) {
    __shared__ int s[TPB / 64];
    unsigned *mask = route_lds;
    int *base = reinterpret_cast<int *>(route_lds + E);
    for (int i = threadIdx.x; i < E; i += TPB) mask[i] = 0u;
    __syncthreads();
    choose<NS>(mu_s, var_s, E, k, 0, T, g_log, o, mask);
    __syncthreads();
    const int total = expert_bases(
        E, [&](int e) { return __popc(mask[e]); }, [](int) { return 0; }, s, base, o.offsets);
    place(k, 0, T, o, mask, base);
    for (int r = total + threadIdx.x; r < T * k; r += TPB) o.token[r] = -1;
}

// counts [blocks][E]: rows of every expert in every workgroup's tokens
template <int NS>
__global__ __launch_bounds__(TPB) void route_choose_kernel(const float *__restrict__ mu_s,
                                                           const float *__restrict__ var_s, int T,
                                                           int E, int k, int g_log, RouteOut o,
                                                           int *__restrict__ counts) {
    unsigned *mask = route_lds;
    for (int i = threadIdx.x; i < E; i += TPB) mask[i] = 0u;
    __syncthreads();
    const int t0 = blockIdx.x * ROUTE_TOKENS;
    choose<NS>(mu_s, var_s, E, k, t0, min(T, t0 + ROUTE_TOKENS), g_log, o, mask);
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += TPB) counts[(size_t)blockIdx.x * E + e] = __popc(mask[e]);
}

// One wave per expert: counts [blocks][E] become the exclusive sums over the workgroups,
// totals [E] the sums.
__global__ __launch_bounds__(64) void route_scan_kernel(int *__restrict__ counts, int blocks,
                                                        int E, int *__restrict__ totals) {
    const int e = blockIdx.x, lane = threadIdx.x;
    int carry = 0;
    for (int b0 = 0; b0 < blocks; b0 += 64) {
        const int b = b0 + lane;
        const int v = b < blocks ? counts[(size_t)b * E + e] : 0;
        int inc = v;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int u = __shfl_up(inc, off, 64);
            if (lane >= off) inc += u;
        }
        if (b < blocks) counts[(size_t)b * E + e] = carry + inc - v;
        carry += __shfl(inc, 63, 64);
    }
    if (lane == 0) totals[e] = carry;
}

__global__ __launch_bounds__(TPB) void route_place_kernel(int T, int E, int k, RouteOut o,
                                                          const int *__restrict__ counts,
                                                          const int *__restrict__ totals) {
    __shared__ int s[TPB / 64];
    unsigned *mask = route_lds;
    int *base = reinterpret_cast<int *>(route_lds + E);
    for (int i = threadIdx.x; i < E; i += TPB) mask[i] = 0u;
    __syncthreads();
    const int t0 = blockIdx.x * ROUTE_TOKENS, t1 = min(T, t0 + ROUTE_TOKENS);
    for (int c = t0 * k + threadIdx.x; c < t1 * k; c += TPB) {
        const int e = o.expert[c];
        if (e >= 0) atomicOr(&mask[e], 1u << (c / k - t0));
    }
    const int total = expert_bases(
        E, [&](int e) { return totals[e]; },
        [&](int e) { return counts[(size_t)blockIdx.x * E + e]; }, s, base,
        blockIdx.x == 0 ? o.offsets : nullptr);
    place(k, t0, t1, o, mask, base);
    // (eight threads per token: their number alone passes 31 bits before T * k does)
    for (long long r = total + (long long)blockIdx.x * TPB + threadIdx.x; r < (long long)T * k;
         r += (long long)gridDim.x * TPB)
        o.token[r] = -1;
}

// ---------------------------------------------------------------------------
// The gated sum, four features of one token per thread. A choice without a row (slot < 0, or a
// slot that is no row) adds nothing.
//   mu_z = sum_j g y,  var_z = sum_j (g^2 + var_g) var_y + var_g y^2
// Bound by memory: 8 bytes per choice and feature in, 8 per feature out. 8192 tokens, 2 choices
// of 4096: 155 us, 5.2 TB/s.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(TPB) void combine_fwd_kernel(
    const float *__restrict__ mu_g, const float *__restrict__ var_g,
    const float *__restrict__ mu_y, const float *__restrict__ var_y, const int *__restrict__ slot,
    int T, int k, int R, int N, bool past_cache, float *__restrict__ mu_z,
    float *__restrict__ var_z) {
    const int groups = (N + 3) / 4;
    const size_t total = (size_t)T * groups, step = (size_t)gridDim.x * TPB;
    for (size_t i = (size_t)blockIdx.x * TPB + threadIdx.x; i < total; i += step) {
        const int t = (int)(i / groups);
        const int g = (int)(i - (size_t)t * groups), valid = in_group(g, N);
        const size_t f = (size_t)g * 4;
        float om[4], ov[4];
#pragma unroll
        for (int c = 0; c < 4; c++) om[c] = ov[c] = 0.f;
        for (int j = 0; j < k; j++) {
            const size_t at = (size_t)t * k + j;
            const int r = slot[at];
            if ((unsigned)r >= (unsigned)R) continue;
            const float gate = mu_g[at], vg = var_g[at], g2 = gate * gate + vg;
            float y[4], v[4];
            load_group(mu_y + (size_t)r * N + f, valid, y);
            load_group(var_y + (size_t)r * N + f, valid, v);
#pragma unroll
            for (int c = 0; c < 4; c++) {
                om[c] += gate * y[c];
                ov[c] += g2 * v[c] + vg * y[c] * y[c];
            }
        }
        store_group(mu_z + (size_t)t * N + f, valid, om, past_cache);
        store_group(var_z + (size_t)t * N + f, valid, ov, past_cache);
    }
}

// Backward, THREADS threads per token:
//   rows    dmu_y = g dmu,  dvar_y = g^2 dvar
//   scores  dmu_s[e] = jcb_g sum_n y dmu,  dvar_s[e] = jcb_g^2 sum_n y^2 dvar;
//           zero for the experts that the token did not choose
// A wave or a workgroup per token, so that its sums stay inside one. Bound by memory: 12 bytes
// per choice and feature (innovations are read once, for further choices from cache), 8 per
// feature. 8192 tokens, 2 choices of 4096: 214 us, 5.0 TB/s.
template <int THREADS>
__global__ __launch_bounds__(TPB) void combine_bwd_kernel(
    const float *__restrict__ mu_g, const float *__restrict__ jcb_g,
    const float *__restrict__ mu_y, const int *__restrict__ expert, const int *__restrict__ slot,
    const float *__restrict__ dmu, const float *__restrict__ dvar, int T, int k, int R, int N,
    int E, bool past_cache, float *__restrict__ dmu_y, float *__restrict__ dvar_y,
    float *__restrict__ dmu_s, float *__restrict__ dvar_s) {
    __shared__ float s[2][TPB / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int x = threadIdx.x % THREADS;
    const int groups = (N + 3) / 4;
    // (whole waves leave the loop, and whole workgroups where it holds a barrier)
    for (long long t = (long long)blockIdx.x * (TPB / THREADS) + threadIdx.x / THREADS; t < T;
         t += (long long)gridDim.x * (TPB / THREADS)) {
        for (int e = x; e < E; e += THREADS) {
            dmu_s[(size_t)t * E + e] = 0.f;
            dvar_s[(size_t)t * E + e] = 0.f;
        }
        for (int j = 0; j < k; j++) {
            const size_t at = (size_t)t * k + j;
            const int r = slot[at], e = expert[at];
            const bool live = (unsigned)r < (unsigned)R;   // the same for all threads of the token
            float sm = 0.f, sv = 0.f;
            if (live) {
                const float g = mu_g[at];
                for (int q = x; q < groups; q += THREADS) {
                    const int valid = in_group(q, N);
                    float y[4], dm[4], dv[4];
                    load_group(mu_y + (size_t)r * N + (size_t)q * 4, valid, y);
                    load_group(dmu + (size_t)t * N + (size_t)q * 4, valid, dm);
                    load_group(dvar + (size_t)t * N + (size_t)q * 4, valid, dv);
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        sm += y[c] * dm[c];
                        sv += y[c] * y[c] * dv[c];
                        dm[c] *= g;
                        dv[c] *= g * g;
                    }
                    store_group(dmu_y + (size_t)r * N + (size_t)q * 4, valid, dm, past_cache);
                    store_group(dvar_y + (size_t)r * N + (size_t)q * 4, valid, dv, past_cache);
                }
            }
#pragma unroll
            for (int off = 32; off > 0; off >>= 1) {
                sm += __shfl_xor(sm, off, 64);
                sv += __shfl_xor(sv, off, 64);
            }
            if (THREADS > 64) {
                if (lane == 0) {
                    s[0][wave] = sm;
                    s[1][wave] = sv;
                }
                __syncthreads();
                sm = (s[0][0] + s[0][1]) + (s[0][2] + s[0][3]);
                sv = (s[1][0] + s[1][1]) + (s[1][2] + s[1][3]);
                __syncthreads();
            }
            // the thread that cleared the entry adds to it, so the accesses stay in order
            if (live && (unsigned)e < (unsigned)E && x == e % THREADS) {
                const float jc = jcb_g[at];
                dmu_s[(size_t)t * E + e] += jc * sm;
                dvar_s[(size_t)t * E + e] += jc * jc * sv;
            }
        }
    }
}

// Rows back to tokens: (sum_j rows[slot] + res) * jcb, jcb^2. Bound by memory. A token's rows
// are few and known, so they are gathered in order and nothing has to be added atomically.
__global__ __launch_bounds__(TPB) void gather_bwd_kernel(
    const float *__restrict__ dmu_r, const float *__restrict__ dvar_r,
    const int *__restrict__ slot, const float *__restrict__ jcb, const float *res_mu,
    const float *res_var, int T, int k, int R, int K, bool past_cache, float *dmu, float *dvar) {
    const int groups = (K + 3) / 4;
    const size_t total = (size_t)T * groups, step = (size_t)gridDim.x * TPB;
    for (size_t i = (size_t)blockIdx.x * TPB + threadIdx.x; i < total; i += step) {
        const int t = (int)(i / groups);
        const int g = (int)(i - (size_t)t * groups), valid = in_group(g, K);
        const size_t f = (size_t)g * 4, at = (size_t)t * K + f;
        float om[4], ov[4];
        if (res_mu != nullptr) {
            load_group(res_mu + at, valid, om);
            load_group(res_var + at, valid, ov);
        } else {
#pragma unroll
            for (int c = 0; c < 4; c++) om[c] = ov[c] = 0.f;
        }
        for (int j = 0; j < k; j++) {
            const int r = slot[(size_t)t * k + j];
            if ((unsigned)r >= (unsigned)R) continue;
            float m[4], v[4];
            load_group(dmu_r + (size_t)r * K + f, valid, m);
            load_group(dvar_r + (size_t)r * K + f, valid, v);
#pragma unroll
            for (int c = 0; c < 4; c++) {
                om[c] += m[c];
                ov[c] += v[c];
            }
        }
        if (jcb != nullptr) {
            float jc[4];
            load_group(jcb + at, valid, jc);
#pragma unroll
            for (int c = 0; c < 4; c++) {
                om[c] *= jc[c];
                ov[c] *= jc[c] * jc[c];
            }
        }
        store_group(dmu + at, valid, om, past_cache);
        store_group(dvar + at, valid, ov, past_cache);
    }
}

// one thread per item up to MAX_BLOCKS workgroups (a launch holds fewer than 2^32 threads),
// which then walk on
constexpr size_t MAX_BLOCKS = (size_t)1 << 22;
inline unsigned blocks_for(size_t n) {
    const size_t b = (n + TPB - 1) / TPB;
    return (unsigned)(b < MAX_BLOCKS ? b : MAX_BLOCKS);
}
inline int route_blocks(int T) { return (T + ROUTE_TOKENS - 1) / ROUTE_TOKENS; }

template <int NS>
hipError_t route(const float *mu_s, const float *var_s, int T, int E, int k, int g_log,
                 const RouteOut &o, int *scratch, hipStream_t stream) {
    const int blocks = route_blocks(T);
    const unsigned lds_mask = E * 4, lds = E * 8;
    if (blocks == 1) {
        hipLaunchKernelGGL(route_one_kernel<NS>, dim3(1), dim3(TPB), lds, stream, mu_s, var_s, T, E,
                           k, g_log, o);
        return hipGetLastError();
    }
    int *totals = scratch, *counts = scratch + E;
    hipLaunchKernelGGL(route_choose_kernel<NS>, dim3(blocks), dim3(TPB), lds_mask, stream, mu_s,
                       var_s, T, E, k, g_log, o, counts);
    hipLaunchKernelGGL(route_scan_kernel, dim3(E), dim3(64), 0, stream, counts, blocks, E, totals);
    hipLaunchKernelGGL(route_place_kernel, dim3(blocks), dim3(TPB), lds, stream, T, E, k, o, counts,
                       totals);
    return hipGetLastError();
}

}  // namespace

size_t moe_route_scratch_ints(int T, int E) {
    return route_blocks(T) > 1 ? ((size_t)route_blocks(T) + 1) * E : 0;
}

hipError_t launch_moe_route(const float *mu_s, const float *var_s, int T, int E, int k, int *expert,
                            float *mu_g, float *var_g, float *jcb_g, int *offsets, int *token,
                            int *slot, int *scratch, hipStream_t stream) {
    const RouteOut o = {expert, mu_g, var_g, jcb_g, offsets, token, slot};
    int g_log = 0;
    while (g_log < 6 && (1 << g_log) < E) g_log++;
    const int ns = (E + 63) / 64;
    if (ns <= 1) return route<1>(mu_s, var_s, T, E, k, g_log, o, scratch, stream);
    if (ns <= 4) return route<4>(mu_s, var_s, T, E, k, g_log, o, scratch, stream);
    return route<16>(mu_s, var_s, T, E, k, g_log, o, scratch, stream);
}

hipError_t launch_moe_combine_fwd(const float *mu_g, const float *var_g, const float *mu_y,
                                  const float *var_y, const int *slot, int T, int k, int R, int N,
                                  float *mu_z, float *var_z, hipStream_t stream) {
    hipLaunchKernelGGL(combine_fwd_kernel, dim3(blocks_for((size_t)T * ((N + 3) / 4))), dim3(TPB), 0,
                       stream, mu_g, var_g, mu_y, var_y, slot, T, k, R, N,
                       goes_past_cache((size_t)2 * T * N), mu_z, var_z);
    return hipGetLastError();
}

hipError_t launch_moe_combine_bwd(const float *mu_g, const float *jcb_g, const float *mu_y,
                                  const int *expert, const int *slot, const float *dmu,
                                  const float *dvar, int T, int k, int R, int N, int E,
                                  float *dmu_y, float *dvar_y, float *dmu_s, float *dvar_s,
                                  hipStream_t stream) {
    const bool past_cache = goes_past_cache((size_t)2 * R * N);
    // a wave per token up to 1024 features, a workgroup beyond
    if (N > 1024)
        hipLaunchKernelGGL(combine_bwd_kernel<256>, dim3(blocks_for((size_t)T * 256)), dim3(TPB), 0, stream,
                           mu_g, jcb_g, mu_y, expert, slot, dmu, dvar, T, k, R, N, E, past_cache, dmu_y,
                           dvar_y, dmu_s, dvar_s);
    else
        hipLaunchKernelGGL(combine_bwd_kernel<64>, dim3(blocks_for((size_t)T * 64)), dim3(TPB), 0, stream,
                           mu_g, jcb_g, mu_y, expert, slot, dmu, dvar, T, k, R, N, E, past_cache, dmu_y,
                           dvar_y, dmu_s, dvar_s);
    return hipGetLastError();
}

hipError_t launch_moe_gather_bwd(const float *dmu_r, const float *dvar_r, const int *slot,
                                 const float *jcb, const float *res_mu, const float *res_var, int T,
                                 int k, int R, int K, float *dmu, float *dvar, hipStream_t stream) {
    hipLaunchKernelGGL(gather_bwd_kernel, dim3(blocks_for((size_t)T * ((K + 3) / 4))), dim3(TPB), 0,
                       stream, dmu_r, dvar_r, slot, jcb, res_mu, res_var, T, k, R, K,
                       goes_past_cache((size_t)2 * T * K), dmu, dvar);
    return hipGetLastError();
}

}  // namespace tagi
