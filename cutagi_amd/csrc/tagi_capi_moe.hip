// C ABI of the layer norm, the Linear layers grouped by expert and the mixture of experts
// (include/tagi_hip.h): argument checks; the launchers choose the kernels.
#include "../../include/tagi_hip.h"
#include "tagi_internal.h"

using namespace tagi;

#define TAGI_TRY(expr)                          \
    do {                                        \
        hipError_t _e = (expr);                 \
        if (_e != hipSuccess) return (int)_e;   \
    } while (0)

namespace {

constexpr int MAX_EXPERTS = 1024, MAX_TOP_K = 64;

hipStream_t as_stream(void *s) { return static_cast<hipStream_t>(s); }

// Sizes that the kernels' indices hold with what is added to them.
constexpr int MAX_SIZE = 1 << 30;

// `columns`: width of the output, `weights`: whether it is [E][N][K]. A launch holds fewer than
// 2^32 threads: the weight backward's kernels have up to 1024 for 32 outputs by 256 inputs, the
// ones for few rows (and for fewer than four inputs or outputs any rows) up to 512 for sixteen
// rows by sixteen columns.
int grouped_sizes(int K, int N, int E, int R, int T, const int *rows, int columns, bool weights) {
    if (K <= 0 || N <= 0 || E <= 0 || R <= 0 || (rows != nullptr && T <= 0))
        return TAGI_ERR_INVALID_ARG;
    if (E > MAX_EXPERTS) return TAGI_ERR_UNSUPPORTED;
    // element offsets of 32 bits inside a tile's 128 rows, and of any row that is gathered
    if (K > (1 << 24) || N > (1 << 24)) return TAGI_ERR_UNSUPPORTED;
    if (rows != nullptr && (long long)T * K > (1LL << 32) - 1) return TAGI_ERR_UNSUPPORTED;
    const double tiles = (columns + 63) / 64 * ((double)R / 64 + E);
    const double weight_wgs = weights ? (double)((K + 255) / 256) * ((N + 31) / 32) * E : 0;
    if (tiles > (1 << 24) - 1 || weight_wgs > (1 << 22) - 1) return TAGI_ERR_UNSUPPORTED;
    const double few = K < 4 || N < 4 ? (columns + 15) / 16 * ((double)R / 16 + E) : 0;
    return few > (1 << 23) - 1 ? TAGI_ERR_UNSUPPORTED : TAGI_OK;
}

int moe_sizes(int T, int k, int R, int N) {
    if (T <= 0 || k <= 0 || R <= 0 || N <= 0) return TAGI_ERR_INVALID_ARG;
    return (long long)T * k > MAX_SIZE || N > MAX_SIZE ? TAGI_ERR_UNSUPPORTED : TAGI_OK;
}

// whether the scratch that a call needs is there, 16-byte aligned
bool scratch_ok(const void *scratch, size_t floats) {
    return scratch != nullptr ? (reinterpret_cast<size_t>(scratch) & 15u) == 0 : floats == 0;
}

int grouped_fwd(const float *mu_w, const float *var_w, const float *mu_b, const float *var_b,
                const float *mu_a, const float *var_a, const int *offsets, const int *rows, int K,
                int N, int E, int R, int T, int bias, int act, void *scratch, float *out0, float *out1,
                float *out2, void *stream) {
    if (!mu_w || !var_w || !mu_a || !var_a || !offsets || !out0 || !out1) return TAGI_ERR_INVALID_ARG;
    if (bias && (!mu_b || !var_b)) return TAGI_ERR_INVALID_ARG;
    const int rc = grouped_sizes(K, N, E, R, T, rows, N, false);
    if (rc != TAGI_OK) return rc;
    if (!scratch_ok(scratch, grouped_scratch_floats(K, N, E, R))) return TAGI_ERR_INVALID_ARG;
    GroupedParams p = {};
    p.x0 = mu_a, p.x1 = var_a, p.y0 = mu_w, p.y1 = var_w;
    p.e0 = bias ? mu_b : nullptr, p.e1 = bias ? var_b : nullptr;
    p.offsets = offsets, p.rows = rows;
    p.K = K, p.N = N, p.E = E, p.R = R, p.T = T, p.act = act;
    p.out0 = out0, p.out1 = out1, p.out2 = out2;
    p.scratch = static_cast<float *>(scratch);
    TAGI_TRY(launch_grouped(GROUPED_FWD, p, as_stream(stream)));
    return TAGI_OK;
}

}  // namespace

extern "C" {

int tagi_layernorm_fwd(const float *mu_w, const float *var_w, const float *mu_b,
                       const float *var_b, const float *mu_a, const float *var_a, int bias,
                       float epsilon, int n, int B, float *mu_s, float *var_s, float *mu_z,
                       float *var_z, void *stream) {
    if (!mu_w || !var_w || !mu_a || !var_a || !mu_s || !var_s || !mu_z || !var_z)
        return TAGI_ERR_INVALID_ARG;
    if (bias && (!mu_b || !var_b)) return TAGI_ERR_INVALID_ARG;
    if (n < 2 || B <= 0) return TAGI_ERR_INVALID_ARG;
    if (n > MAX_SIZE || B > MAX_SIZE) return TAGI_ERR_UNSUPPORTED;
    TAGI_TRY(launch_layernorm_fwd(mu_w, var_w, bias ? mu_b : nullptr, bias ? var_b : nullptr, mu_a,
                                  var_a, epsilon, n, B, mu_s, var_s, mu_z, var_z,
                                  as_stream(stream)));
    return TAGI_OK;
}

int tagi_layernorm_bwd_scratch(int n, int B, size_t *bytes) {
    if (bytes == nullptr || n < 2 || B <= 0) return TAGI_ERR_INVALID_ARG;
    if (n > MAX_SIZE || B > MAX_SIZE) return TAGI_ERR_UNSUPPORTED;
    *bytes = layernorm_bwd_scratch_floats(n, B) * sizeof(float);
    return TAGI_OK;
}

int tagi_layernorm_bwd(const float *mu_w, const float *var_w, const float *var_b,
                       const float *mu_a, const float *jcb, const float *mu_s, const float *var_s,
                       const float *delta_mu_out, const float *delta_var_out, float epsilon, int n,
                       int B, int bias, int state_update, int param_update, void *scratch,
                       float *delta_mu, float *delta_var, float *delta_mu_w, float *delta_var_w,
                       float *delta_mu_b, float *delta_var_b, void *stream) {
    if (!mu_w || !var_w || !mu_s || !var_s || !delta_mu_out || !delta_var_out)
        return TAGI_ERR_INVALID_ARG;
    if (state_update && (!delta_mu || !delta_var)) return TAGI_ERR_INVALID_ARG;
    if (param_update && (!mu_a || !delta_mu_w || !delta_var_w)) return TAGI_ERR_INVALID_ARG;
    if (param_update && bias && (!var_b || !delta_mu_b || !delta_var_b))
        return TAGI_ERR_INVALID_ARG;
    if (n < 2 || B <= 0) return TAGI_ERR_INVALID_ARG;
    if (n > MAX_SIZE || B > MAX_SIZE) return TAGI_ERR_UNSUPPORTED;
    if (!state_update && !param_update) return TAGI_OK;
    if (param_update && !scratch_ok(scratch, layernorm_bwd_scratch_floats(n, B))) return TAGI_ERR_INVALID_ARG;
    TAGI_TRY(launch_layernorm_bwd(mu_w, var_w, bias ? var_b : nullptr, mu_a, jcb, mu_s, var_s,
                                  delta_mu_out, delta_var_out, epsilon, n, B, state_update,
                                  param_update, static_cast<float *>(scratch), delta_mu, delta_var,
                                  delta_mu_w, delta_var_w, delta_mu_b, delta_var_b,
                                  as_stream(stream)));
    return TAGI_OK;
}

int tagi_grouped_linear_scratch(int K, int N, int E, int R, size_t *bytes) {
    if (bytes == nullptr) return TAGI_ERR_INVALID_ARG;
    const int rc = grouped_sizes(K, N, E, R, 0, nullptr, N, false);
    if (rc != TAGI_OK) return rc;
    *bytes = grouped_scratch_floats(K, N, E, R) * sizeof(float);
    return TAGI_OK;
}

int tagi_grouped_linear_fwd(const float *mu_w, const float *var_w, const float *mu_b,
                            const float *var_b, const float *mu_a, const float *var_a,
                            const int *offsets, const int *rows, int K, int N, int E, int R, int T,
                            int bias, void *scratch, float *mu_z, float *var_z, void *stream) {
    return grouped_fwd(mu_w, var_w, mu_b, var_b, mu_a, var_a, offsets, rows, K, N, E, R, T, bias, 0,
                       scratch, mu_z, var_z, nullptr, stream);
}

int tagi_grouped_linear_fwd_act(const float *mu_w, const float *var_w, const float *mu_b,
                                const float *var_b, const float *mu_a, const float *var_a,
                                const int *offsets, const int *rows, int K, int N, int E, int R,
                                int T, int bias, int activation, void *scratch, float *mu_out,
                                float *var_out, float *jcb_out, void *stream) {
    if (activation != TAGI_ACT_RELU && activation != TAGI_ACT_MIXTURE_RELU)
        return TAGI_ERR_INVALID_ARG;
    if (!jcb_out) return TAGI_ERR_INVALID_ARG;
    return grouped_fwd(mu_w, var_w, mu_b, var_b, mu_a, var_a, offsets, rows, K, N, E, R, T, bias,
                       activation, scratch, mu_out, var_out, jcb_out, stream);
}

int tagi_grouped_linear_bwd(const float *mu_w, const float *var_w, const float *var_b,
                            const float *mu_a, const float *jcb, const float *delta_mu,
                            const float *delta_var, const int *offsets, const int *rows, int K,
                            int N, int E, int R, int T, int bias, int state_update,
                            int param_update, void *scratch, float *delta_mu_z,
                            float *delta_var_z, float *delta_mu_w, float *delta_var_w,
                            float *delta_mu_b, float *delta_var_b, void *stream) {
    if (!delta_mu || !delta_var || !offsets) return TAGI_ERR_INVALID_ARG;
    if (state_update && (!mu_w || !delta_mu_z || !delta_var_z)) return TAGI_ERR_INVALID_ARG;
    if (param_update && (!var_w || !mu_a || !delta_mu_w || !delta_var_w))
        return TAGI_ERR_INVALID_ARG;
    if (param_update && bias && (!var_b || !delta_mu_b || !delta_var_b))
        return TAGI_ERR_INVALID_ARG;
    const int rc = grouped_sizes(K, N, E, R, T, rows, K, param_update != 0);
    if (rc != TAGI_OK) return rc;
    if (!scratch_ok(scratch, grouped_scratch_floats(K, N, E, R))) return TAGI_ERR_INVALID_ARG;
    GroupedParams p = {};
    p.scratch = static_cast<float *>(scratch);
    p.x0 = delta_mu, p.x1 = delta_var;
    p.offsets = offsets, p.rows = rows;
    p.K = K, p.N = N, p.E = E, p.R = R, p.T = T;
    if (state_update) {
        p.y0 = mu_w, p.e0 = jcb, p.out0 = delta_mu_z, p.out1 = delta_var_z;
        TAGI_TRY(launch_grouped(GROUPED_DZ, p, as_stream(stream)));
    }
    if (param_update) {
        p.y0 = mu_a, p.e0 = var_w, p.out0 = delta_mu_w, p.out1 = delta_var_w;
        if (bias) p.e1 = var_b, p.db0 = delta_mu_b, p.db1 = delta_var_b;
        TAGI_TRY(launch_grouped(GROUPED_DW, p, as_stream(stream)));
    }
    return TAGI_OK;
}

int tagi_moe_route_scratch(int T, int E, size_t *bytes) {
    if (bytes == nullptr || T <= 0 || E <= 0) return TAGI_ERR_INVALID_ARG;
    if (E > MAX_EXPERTS) return TAGI_ERR_UNSUPPORTED;
    *bytes = moe_route_scratch_ints(T, E) * sizeof(int);
    return TAGI_OK;
}

int tagi_moe_route(const float *mu_s, const float *var_s, int T, int E, int top_k, void *scratch,
                   int *expert, float *mu_g, float *var_g, float *jcb_g, int *offsets, int *token,
                   int *slot, void *stream) {
    if (!mu_s || !var_s || !expert || !mu_g || !var_g || !jcb_g || !offsets || !token || !slot)
        return TAGI_ERR_INVALID_ARG;
    if (T <= 0 || E <= 0 || top_k <= 0 || top_k > E) return TAGI_ERR_INVALID_ARG;
    // (32 tokens to a workgroup of 256 threads, and a launch holds fewer than 2^32 of them)
    if (E > MAX_EXPERTS || top_k > MAX_TOP_K || (long long)T * top_k > MAX_SIZE || T > (1 << 29) - 32)
        return TAGI_ERR_UNSUPPORTED;
    if (moe_route_scratch_ints(T, E) > 0 && !scratch) return TAGI_ERR_INVALID_ARG;
    TAGI_TRY(launch_moe_route(mu_s, var_s, T, E, top_k, expert, mu_g, var_g, jcb_g, offsets, token,
                              slot, static_cast<int *>(scratch), as_stream(stream)));
    return TAGI_OK;
}

int tagi_moe_combine_fwd(const float *mu_g, const float *var_g, const float *mu_y,
                         const float *var_y, const int *slot, int T, int top_k, int R, int N,
                         float *mu_z, float *var_z, void *stream) {
    if (!mu_g || !var_g || !mu_y || !var_y || !slot || !mu_z || !var_z) return TAGI_ERR_INVALID_ARG;
    const int rc = moe_sizes(T, top_k, R, N);
    if (rc != TAGI_OK) return rc;
    TAGI_TRY(launch_moe_combine_fwd(mu_g, var_g, mu_y, var_y, slot, T, top_k, R, N, mu_z, var_z,
                                    as_stream(stream)));
    return TAGI_OK;
}

int tagi_moe_combine_bwd(const float *mu_g, const float *jcb_g, const float *mu_y,
                         const int *expert, const int *slot, const float *delta_mu,
                         const float *delta_var, int T, int top_k, int R, int N, int E,
                         float *delta_mu_y, float *delta_var_y, float *delta_mu_s,
                         float *delta_var_s, void *stream) {
    if (!mu_g || !jcb_g || !mu_y || !expert || !slot || !delta_mu || !delta_var || !delta_mu_y ||
        !delta_var_y || !delta_mu_s || !delta_var_s)
        return TAGI_ERR_INVALID_ARG;
    const int rc = moe_sizes(T, top_k, R, N);
    if (rc != TAGI_OK) return rc;
    if (E <= 0) return TAGI_ERR_INVALID_ARG;
    if (E > MAX_SIZE) return TAGI_ERR_UNSUPPORTED;
    TAGI_TRY(launch_moe_combine_bwd(mu_g, jcb_g, mu_y, expert, slot, delta_mu, delta_var, T, top_k,
                                    R, N, E, delta_mu_y, delta_var_y, delta_mu_s, delta_var_s,
                                    as_stream(stream)));
    return TAGI_OK;
}

int tagi_moe_gather_bwd(const float *delta_mu_r, const float *delta_var_r, const int *slot,
                        const float *jcb, const float *res_mu, const float *res_var, int T,
                        int top_k, int R, int K, float *delta_mu, float *delta_var, void *stream) {
    if (!delta_mu_r || !delta_var_r || !slot || !delta_mu || !delta_var) return TAGI_ERR_INVALID_ARG;
    if ((res_mu == nullptr) != (res_var == nullptr)) return TAGI_ERR_INVALID_ARG;
    const int rc = moe_sizes(T, top_k, R, K);
    if (rc != TAGI_OK) return rc;
    TAGI_TRY(launch_moe_gather_bwd(delta_mu_r, delta_var_r, slot, jcb, res_mu, res_var, T, top_k, R,
                                   K, delta_mu, delta_var, as_stream(stream)));
    return TAGI_OK;
}

}  // extern "C"
