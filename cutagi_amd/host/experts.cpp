// LayerNorm and MixtureOfExperts: see experts.h.
#include "experts.h"

#include <algorithm>
#include <cmath>

#include "../../include/tagi_hip.h"
#include "host_util.h"
#include "logger.h"

namespace tagi_host {

// ---- LayerNorm -------------------------------------------------------------------------
namespace {
size_t features_of(const std::vector<int> &shape) {
    size_t n = shape.empty() ? 0 : 1;
    for (int s : shape) n *= s > 0 ? (size_t)s : 0;
    if (n < 2)
        LOG(LogLevel::ERROR, "LayerNorm needs a normalized shape of two features or more");
    return n;
}
// as the other normalisation layers: weights start at one, biases at zero, variances at
// 2 / (in + out) * gain^2
void init_layernorm(BaseLayer &l, float gain_w, float gain_b) {
    const size_t n = l.input_size;
    const float scale = 2.0f / (float)(n + n);
    l.num_weights = n;
    l.num_biases = l.bias ? n : 0;
    l.mu_w.assign(n, 1.0f);
    l.var_w.assign(n, scale * gain_w * gain_w);
    l.mu_b.assign(l.num_biases, 0.0f);
    l.var_b.assign(l.num_biases, scale * gain_b * gain_b);
}
}  // namespace

LayerNorm::LayerNorm(const std::vector<int> &shape, float eps, bool bias, float gain_weight,
                     float gain_bias, int device_idx)
    : normalized_shape(shape), epsilon(eps), gain_w(gain_weight), gain_b(gain_bias) {
    this->input_size = this->output_size = features_of(shape);
    this->bias = bias;
    this->device_idx = device_idx;
    this->init_weight_bias();
    if (this->training) this->allocate_param_delta();
}

void LayerNorm::init_weight_bias() { init_layernorm(*this, gain_w, gain_b); }

std::unique_ptr<BaseLayer> LayerNorm::to_cuda(int device_idx) {
    this->device = "cuda";
    this->device_idx = device_idx;
    auto layer = std::make_unique<LayerNormHip>(normalized_shape, epsilon, bias, gain_w, gain_b,
                                                device_idx);
    layer->copy_params_from(*this);
    return layer;
}

LayerNormHip::LayerNormHip(const std::vector<int> &shape, float eps, bool bias, float gain_weight,
                           float gain_bias, int device_idx)
    : normalized_shape(shape), epsilon(eps), gain_w(gain_weight), gain_b(gain_bias) {
    this->input_size = this->output_size = features_of(shape);
    this->bias = bias;
    this->device_idx = device_idx;
    this->num_weights = this->input_size;
    this->num_biases = bias ? this->input_size : 0;
    if (this->training) this->allocate_param_delta();
}

LayerNormHip::~LayerNormHip() {
    dev_free_t(d_mu_s);
    dev_free_t(d_var_s);
    dev_free_t(d_scratch);
}

void LayerNormHip::init_weight_bias() {
    init_layernorm(*this, gain_w, gain_b);
    this->allocate_param_memory();
    this->params_to_device();
}

void LayerNormHip::hold(int batch_size) {
    if ((size_t)batch_size > rows_held) {
        freed += d_mu_s != nullptr;
        dev_free_t(d_mu_s);
        dev_free_t(d_var_s);
        rows_held = 0;
        d_mu_s = dev_alloc_t<float>(batch_size, device_idx);
        d_var_s = dev_alloc_t<float>(batch_size, device_idx);
        rows_held = batch_size;
    }
    if (!training) return;
    // the backward pass's scratch memory too: the recording of a pass allocates nothing
    size_t bytes = 0;
    TAGI_OK_OR_THROW(tagi_layernorm_bwd_scratch((int)input_size, batch_size, &bytes));
    if (bytes > scratch_held) {
        freed += d_scratch != nullptr;
        dev_free_t(d_scratch);
        scratch_held = 0;
        d_scratch = dev_alloc_t<char>(bytes, device_idx);
        scratch_held = bytes;
    }
}

void LayerNormHip::forward_replayed(int batch_size) {
    BaseLayerHip::forward_replayed(batch_size);
    trained_batch = training ? batch_size : 0;
}

// reference: LayerNormCuda::forward, src/layernorm_layer_cuda.cu
void LayerNormHip::forward(BaseHiddenStates &input_states, BaseHiddenStates &output_states,
                           BaseTempStates &) {
    auto *in = as<HiddenStateHip>(input_states);
    auto *out = as<HiddenStateHip>(output_states);
    const int batch_size = (int)input_states.block_size;
    this->set_cap_factor_udapte(batch_size);
    if (this->input_size != input_states.actual_size)
        LOG(LogLevel::ERROR, "Input size mismatch: " + std::to_string(this->input_size) + " vs " +
                                 std::to_string(input_states.actual_size));
    if (this->output_size * batch_size > out->size)
        LOG(LogLevel::ERROR, "Output state buffer too small for " + this->get_layer_info());
    this->require_params(input_size, input_size);
    this->hold(batch_size);
    TAGI_OK_OR_THROW(tagi_layernorm_fwd(d_mu_w, d_var_w, d_mu_b, d_var_b, in->d_mu_a, in->d_var_a,
                                        bias ? 1 : 0, epsilon, (int)input_size, batch_size, d_mu_s,
                                        d_var_s, out->d_mu_a, out->d_var_a, host_stream()));
    output_states.width = this->out_width;
    output_states.height = this->out_height;
    output_states.depth = this->out_channels;
    output_states.block_size = batch_size;
    output_states.actual_size = this->output_size;
    trained_batch = training ? batch_size : 0;
    out->jcb_ones = true;
    if (this->training) this->store_states_for_training_hip(*in, *out);
}

// reference: LayerNormCuda::backward, src/layernorm_layer_cuda.cu
void LayerNormHip::backward(BaseDeltaStates &input_delta_states, BaseDeltaStates &output_delta_states,
                            BaseTempStates &, bool state_udapte) {
    auto *din = as<DeltaStateHip>(input_delta_states);
    auto *dout = as<DeltaStateHip>(output_delta_states);
    auto *bwd = dynamic_cast<BackwardStateHip *>(this->bwd_states.get());
    const int batch_size = (int)input_delta_states.block_size;
    if (state_udapte && input_size * batch_size > dout->size)
        LOG(LogLevel::ERROR, "Delta state buffer too small for " + this->get_layer_info());
    if (batch_size > trained_batch || bwd->d_mu_a == nullptr)
        LOG(LogLevel::ERROR, "Backward pass of " + this->get_layer_info() + " without its forward pass in training mode");
    TAGI_OK_OR_THROW(tagi_layernorm_bwd(
        d_mu_w, d_var_w, d_var_b, bwd->d_mu_a, bwd->jcb_ones ? nullptr : bwd->d_jcb, d_mu_s, d_var_s,
        din->d_delta_mu, din->d_delta_var, epsilon, (int)input_size, batch_size, bias ? 1 : 0,
        state_udapte ? 1 : 0, param_update ? 1 : 0, d_scratch, dout->d_delta_mu, dout->d_delta_var,
        d_delta_mu_w, d_delta_var_w, d_delta_mu_b, d_delta_var_b, host_stream()));
}

// ---- MixtureOfExperts --------------------------------------------------------------------
std::string MoeSizes::info() const {
    return "MixtureOfExperts(" + std::to_string(input) + "," + std::to_string(hidden) + "," +
           std::to_string(output) + "," + std::to_string(experts) + "," + std::to_string(top_k) + ")";
}

namespace {
MoeSizes moe_sizes(size_t input, size_t hidden, size_t output, int experts, int top_k,
                   const std::string &activation) {
    MoeSizes s;
    if (input == 0 || hidden == 0 || output == 0)
        LOG(LogLevel::ERROR, "MixtureOfExperts needs sizes of one or more");
    if (experts < 1 || experts > 1024)
        LOG(LogLevel::ERROR, "MixtureOfExperts takes 1 to 1024 experts");
    if (top_k < 1 || top_k > experts || top_k > 64)
        LOG(LogLevel::ERROR, "MixtureOfExperts: top_k is 1 to the number of experts, 64 at most");
    if (activation == "relu")
        s.activation = TAGI_ACT_RELU;
    else if (activation == "mixture_relu")
        s.activation = TAGI_ACT_MIXTURE_RELU;
    else
        LOG(LogLevel::ERROR, "MixtureOfExperts: activation [" + activation + "] is not supported.");
    s.input = input;
    s.hidden = hidden;
    s.output = output;
    s.experts = experts;
    s.top_k = top_k;
    return s;
}

// every part starts like a Linear layer of its sizes
void init_moe(BaseLayer &l, const MoeSizes &s, float gain_w, float gain_b, const std::string &method) {
    l.mu_w.clear(), l.var_w.clear(), l.mu_b.clear(), l.var_b.clear();
    auto part = [&](size_t in, size_t out, size_t count) {
        const ParameterTuple p = init_gaussian_params(method, gain_w, gain_b, (float)in, (float)out,
                                                      count * in * out, l.bias ? count * out : 0);
        auto add = [](std::vector<float> &to, const std::vector<float> &from) {
            to.insert(to.end(), from.begin(), from.end());
        };
        add(l.mu_w, std::get<0>(p));
        add(l.var_w, std::get<1>(p));
        add(l.mu_b, std::get<2>(p));
        add(l.var_b, std::get<3>(p));
    };
    part(s.input, s.experts, 1);
    part(s.input, s.hidden, s.experts);
    part(s.hidden, s.output, s.experts);
    l.num_weights = l.mu_w.size();
    l.num_biases = l.mu_b.size();
}
}  // namespace

MixtureOfExperts::MixtureOfExperts(size_t input_size, size_t hidden_size, size_t output_size,
                                   int num_experts, int top_k, const std::string &activation,
                                   bool bias, float gain_weight, float gain_bias, std::string method,
                                   int device_idx)
    : sizes(moe_sizes(input_size, hidden_size, output_size, num_experts, top_k, activation)),
      gain_w(gain_weight), gain_b(gain_bias), init_method(std::move(method)) {
    this->input_size = input_size;
    this->output_size = output_size;
    this->bias = bias;
    this->device_idx = device_idx;
    this->init_weight_bias();
    if (this->training) this->allocate_param_delta();
}

void MixtureOfExperts::init_weight_bias() { init_moe(*this, sizes, gain_w, gain_b, init_method); }

std::unique_ptr<BaseLayer> MixtureOfExperts::to_cuda(int device_idx) {
    this->device = "cuda";
    this->device_idx = device_idx;
    auto layer = std::make_unique<MixtureOfExpertsHip>(sizes, bias, gain_w, gain_b, init_method, device_idx);
    layer->copy_params_from(*this);
    return layer;
}

MixtureOfExpertsHip::MixtureOfExpertsHip(const MoeSizes &s, bool bias, float gain_weight,
                                         float gain_bias, std::string method, int device_idx)
    : sizes(s), gain_w(gain_weight), gain_b(gain_bias), init_method(std::move(method)) {
    this->input_size = s.input;
    this->output_size = s.output;
    this->bias = bias;
    this->device_idx = device_idx;
    this->num_weights = s.weights();
    this->num_biases = bias ? s.biases() : 0;
    if (this->training) this->allocate_param_delta();
}

MixtureOfExpertsHip::~MixtureOfExpertsHip() { dev_free_t(d_work); }

void MixtureOfExpertsHip::init_weight_bias() {
    init_moe(*this, sizes, gain_w, gain_b, init_method);
    this->allocate_param_memory();
    this->params_to_device();
}

// Pointers into d_work for a batch (null pointers where d_work is null: then `bytes` is the
// size that the batch needs).
struct MixtureOfExpertsHip::Work {
    int *expert, *slot, *token, *offsets;   // [T][k], [T][k], [T k], [E + 1]
    float *mu_g, *var_g, *jcb_g;            // [T][k]
    float *mu_s, *var_s, *dmu_s, *dvar_s;   // [T][E] scores and their innovations
    float *mu_h, *var_h, *jcb_h;            // [T k][hidden]
    float *mu_y, *var_y;                    // [T k][output]
    float *dmu_y, *dvar_y;                  // [T k][output]
    float *dmu_h, *dvar_h;                  // [T k][hidden]
    float *dmu_x, *dvar_x;                  // [T k][input]
    void *scratch;                          // of one call at a time
    size_t bytes;
};

MixtureOfExpertsHip::Work MixtureOfExpertsHip::work(int batch) const {
    const size_t T = batch, E = sizes.experts, R = T * sizes.top_k;
    Work w;
    size_t at = 0;
    auto take = [&](auto *&p, size_t n) {
        using V = std::remove_pointer_t<std::remove_reference_t<decltype(p)>>;
        p = d_work == nullptr ? nullptr : reinterpret_cast<V *>(d_work + at);
        at += (n * 4 + 255) / 256 * 256;
    };
    take(w.expert, R), take(w.slot, R), take(w.token, R), take(w.offsets, E + 1);
    take(w.mu_g, R), take(w.var_g, R), take(w.jcb_g, R);
    take(w.mu_s, T * E), take(w.var_s, T * E), take(w.dmu_s, T * E), take(w.dvar_s, T * E);
    take(w.mu_h, R * sizes.hidden), take(w.var_h, R * sizes.hidden), take(w.jcb_h, R * sizes.hidden);
    take(w.mu_y, R * sizes.output), take(w.var_y, R * sizes.output);
    take(w.dmu_y, R * sizes.output), take(w.dvar_y, R * sizes.output);
    take(w.dmu_h, R * sizes.hidden), take(w.dvar_h, R * sizes.hidden);
    take(w.dmu_x, R * sizes.input), take(w.dvar_x, R * sizes.input);
    const int K = (int)sizes.input, H = (int)sizes.hidden, N = (int)sizes.output;
    size_t scratch = 0, up = 0, down = 0;
    TAGI_OK_OR_THROW(tagi_moe_route_scratch(batch, sizes.experts, &scratch));
    TAGI_OK_OR_THROW(tagi_grouped_linear_scratch(K, H, sizes.experts, (int)R, &up));
    TAGI_OK_OR_THROW(tagi_grouped_linear_scratch(H, N, sizes.experts, (int)R, &down));
    scratch = std::max(scratch, std::max(up, down));
    char *s = nullptr;
    take(s, (scratch + 3) / 4);
    w.scratch = s;
    w.bytes = at;
    return w;
}

void MixtureOfExpertsHip::hold(int batch) {
    if ((size_t)batch <= batch_held) return;
    freed += d_work != nullptr;
    dev_free_t(d_work);
    batch_held = 0;
    const size_t bytes = this->work(batch).bytes;
    d_work = dev_alloc_t<char>(bytes, device_idx);
    batch_held = batch;
}

void MixtureOfExpertsHip::forward(BaseHiddenStates &input_states, BaseHiddenStates &output_states,
                                  BaseTempStates &) {
    auto *in = as<HiddenStateHip>(input_states);
    auto *out = as<HiddenStateHip>(output_states);
    const int T = (int)input_states.block_size;
    this->set_cap_factor_udapte(T);
    if (this->input_size != input_states.actual_size)
        LOG(LogLevel::ERROR, "Input size mismatch: " + std::to_string(this->input_size) + " vs " +
                                 std::to_string(input_states.actual_size));
    if (this->output_size * T > out->size)
        LOG(LogLevel::ERROR, "Output state buffer too small for " + this->get_layer_info());
    this->require_params(sizes.weights(), sizes.biases());
    this->hold(T);
    const Work w = this->work(T);
    const int K = (int)sizes.input, H = (int)sizes.hidden, N = (int)sizes.output;
    const int E = sizes.experts, k = sizes.top_k, R = T * k, has_b = bias ? 1 : 0;
    const size_t up = sizes.router_weights(), down = up + sizes.up_weights();
    const size_t up_b = E, down_b = up_b + (size_t)E * H;
    auto b = [&](const float *p, size_t at) { return bias ? p + at : nullptr; };
    void *stream = host_stream();

    TAGI_OK_OR_THROW(tagi_linear_fwd(d_mu_w, d_var_w, b(d_mu_b, 0), b(d_var_b, 0), in->d_mu_a,
                                     in->d_var_a, K, E, T, has_b, w.mu_s, w.var_s, stream));
    TAGI_OK_OR_THROW(tagi_moe_route(w.mu_s, w.var_s, T, E, k, w.scratch, w.expert, w.mu_g, w.var_g,
                                    w.jcb_g, w.offsets, w.token, w.slot, stream));
    TAGI_OK_OR_THROW(tagi_grouped_linear_fwd_act(
        d_mu_w + up, d_var_w + up, b(d_mu_b, up_b), b(d_var_b, up_b), in->d_mu_a, in->d_var_a,
        w.offsets, w.token, K, H, E, R, T, has_b, sizes.activation, w.scratch, w.mu_h, w.var_h,
        w.jcb_h, stream));
    TAGI_OK_OR_THROW(tagi_grouped_linear_fwd(
        d_mu_w + down, d_var_w + down, b(d_mu_b, down_b), b(d_var_b, down_b), w.mu_h, w.var_h,
        w.offsets, nullptr, H, N, E, R, R, has_b, w.scratch, w.mu_y, w.var_y, stream));
    TAGI_OK_OR_THROW(tagi_moe_combine_fwd(w.mu_g, w.var_g, w.mu_y, w.var_y, w.slot, T, k, R, N,
                                          out->d_mu_a, out->d_var_a, stream));
    last_batch = T;
    trained_batch = training ? T : 0;
    output_states.width = this->out_width;
    output_states.height = this->out_height;
    output_states.depth = this->out_channels;
    output_states.block_size = T;
    output_states.actual_size = this->output_size;
    out->jcb_ones = true;
    if (this->training) this->store_states_for_training_hip(*in, *out);
}

void MixtureOfExpertsHip::backward(BaseDeltaStates &input_delta_states,
                                   BaseDeltaStates &output_delta_states, BaseTempStates &,
                                   bool state_udapte) {
    auto *din = as<DeltaStateHip>(input_delta_states);
    auto *dout = as<DeltaStateHip>(output_delta_states);
    auto *bwd = dynamic_cast<BackwardStateHip *>(this->bwd_states.get());
    const int T = (int)input_delta_states.block_size;
    if (state_udapte && input_size * T > dout->size)
        LOG(LogLevel::ERROR, "Delta state buffer too small for " + this->get_layer_info());
    if (T != trained_batch || bwd->d_mu_a == nullptr)
        LOG(LogLevel::ERROR, "Backward pass of " + this->get_layer_info() + " without its forward pass in training mode");
    const Work w = this->work(T);
    const int K = (int)sizes.input, H = (int)sizes.hidden, N = (int)sizes.output;
    const int E = sizes.experts, k = sizes.top_k, R = T * k, has_b = bias ? 1 : 0;
    const size_t up = sizes.router_weights(), down = up + sizes.up_weights();
    const size_t up_b = E, down_b = up_b + (size_t)E * H;
    auto b = [&](float *p, size_t at) { return bias ? p + at : nullptr; };
    const int params = param_update ? 1 : 0, states = state_udapte ? 1 : 0;
    void *stream = host_stream();

    TAGI_OK_OR_THROW(tagi_moe_combine_bwd(w.mu_g, w.jcb_g, w.mu_y, w.expert, w.slot, din->d_delta_mu,
                                          din->d_delta_var, T, k, R, N, E, w.dmu_y, w.dvar_y, w.dmu_s,
                                          w.dvar_s, stream));
    TAGI_OK_OR_THROW(tagi_grouped_linear_bwd(
        d_mu_w + down, d_var_w + down, b(d_var_b, down_b), w.mu_h, w.jcb_h, w.dmu_y, w.dvar_y, w.offsets,
        nullptr, H, N, E, R, R, has_b, 1, params, w.scratch, w.dmu_h, w.dvar_h, d_delta_mu_w + down,
        d_delta_var_w + down, b(d_delta_mu_b, down_b), b(d_delta_var_b, down_b), stream));
    if (states || params)
        TAGI_OK_OR_THROW(tagi_grouped_linear_bwd(
            d_mu_w + up, d_var_w + up, b(d_var_b, up_b), bwd->d_mu_a, nullptr, w.dmu_h, w.dvar_h,
            w.offsets, w.token, K, H, E, R, T, has_b, states, params, w.scratch, w.dmu_x, w.dvar_x,
            d_delta_mu_w + up, d_delta_var_w + up, b(d_delta_mu_b, up_b), b(d_delta_var_b, up_b), stream));
    // the router's share of the state innovations, not yet times the Jacobian, then both
    TAGI_OK_OR_THROW(tagi_linear_bwd(
        d_mu_w, d_var_w, b(d_var_b, 0), bwd->d_mu_a, device_ones(bwd->size, device_idx), w.dmu_s,
        w.dvar_s, K, E, T, has_b, states, params, dout->d_delta_mu, dout->d_delta_var, d_delta_mu_w,
        d_delta_var_w, b(d_delta_mu_b, 0), b(d_delta_var_b, 0), stream));
    if (states)
        TAGI_OK_OR_THROW(tagi_moe_gather_bwd(w.dmu_x, w.dvar_x, w.slot,
                                             bwd->jcb_ones ? nullptr : bwd->d_jcb, dout->d_delta_mu,
                                             dout->d_delta_var, T, k, R, K, dout->d_delta_mu,
                                             dout->d_delta_var, stream));
}

void MixtureOfExpertsHip::forward_replayed(int batch_size) {
    BaseLayerHip::forward_replayed(batch_size);
    last_batch = batch_size;
    trained_batch = training ? batch_size : 0;
}

std::vector<int> MixtureOfExpertsHip::get_expert_choices() {
    std::vector<int> v((size_t)last_batch * sizes.top_k);
    if (v.empty()) return v;
    HIP_OK(hipStreamSynchronize(host_stream()));
    HIP_OK(hipMemcpy(v.data(), this->work(last_batch).expert, v.size() * sizeof(int), hipMemcpyDeviceToHost));
    return v;
}

}  // namespace tagi_host
