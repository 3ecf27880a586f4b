// The layers of a mixture-of-experts feed-forward block, each with the device form that
// to_cuda() returns: LayerNorm (reference: include/layernorm_layer.h), normalisation over the
// features of each sample, and MixtureOfExperts (no counterpart in the reference): a router
// that sends every sample to top_k of num_experts two-layer perceptrons and adds their outputs
// up, weighted by its gates. As for every layer here, the host forms only hold configuration
// and parameters; all arithmetic runs on the GPU behind the C ABI.
#pragma once
#include <memory>
#include <string>
#include <vector>

#include "layers.h"

namespace tagi_host {

// ---- LayerNorm -------------------------------------------------------------------------
class LayerNorm : public BaseLayer {
   public:
    std::vector<int> normalized_shape;
    float epsilon, gain_w, gain_b;

    LayerNorm(const std::vector<int> &normalized_shape, float eps = 1e-5f, bool bias = true,
              float gain_weight = 1.0f, float gain_bias = 1.0f, int device_idx = 0);
    std::string get_layer_info() const override { return "LayerNorm()"; }
    std::string get_layer_name() const override { return "LayerNorm"; }
    LayerType get_layer_type() const override { return LayerType::Norm; }
    void init_weight_bias() override;
    std::unique_ptr<BaseLayer> to_cuda(int device_idx = 0) override;
};

class LayerNormHip : public BaseLayerHip {
   public:
    std::vector<int> normalized_shape;
    float epsilon, gain_w, gain_b;

    LayerNormHip(const std::vector<int> &normalized_shape, float eps = 1e-5f, bool bias = true,
                 float gain_weight = 1.0f, float gain_bias = 1.0f, int device_idx = 0);
    ~LayerNormHip() override;
    std::string get_layer_info() const override { return "LayerNorm()"; }
    std::string get_layer_name() const override { return "LayerNormCuda"; }
    LayerType get_layer_type() const override { return LayerType::Norm; }
    void init_weight_bias() override;
    void forward(BaseHiddenStates &input_states, BaseHiddenStates &output_states,
                 BaseTempStates &temp_states) override;
    void backward(BaseDeltaStates &input_delta_states, BaseDeltaStates &output_delta_states,
                  BaseTempStates &temp_states, bool state_udapte = true) override;
    void forward_replayed(int batch_size) override;

   private:
    // rows that the backward pass finds: those of the last forward pass, none if that was an
    // evaluation (whose statistics have taken their place)
    int trained_batch = 0;
    // statistics of the rows of the last forward pass, sums of the backward pass; as large as
    // the largest batch seen (in training) needs
    float *d_mu_s = nullptr, *d_var_s = nullptr;
    char *d_scratch = nullptr;
    size_t rows_held = 0, scratch_held = 0;
    void hold(int batch_size);
};

// ---- MixtureOfExperts --------------------------------------------------------------------
// Parameters, one after the other in the layer's weights: router [experts][input], first
// layers [experts][hidden][input], second layers [experts][output][hidden]; biases likewise.
struct MoeSizes {
    size_t input = 0, hidden = 0, output = 0;
    int experts = 0, top_k = 0;
    int activation = TAGI_ACT_RELU;   // between the two layers of an expert
    size_t router_weights() const { return (size_t)experts * input; }
    size_t up_weights() const { return (size_t)experts * hidden * input; }
    size_t down_weights() const { return (size_t)experts * output * hidden; }
    size_t weights() const { return router_weights() + up_weights() + down_weights(); }
    size_t biases() const { return (size_t)experts * (1 + hidden + output); }
    std::string info() const;
};

class MixtureOfExperts : public BaseLayer {
   public:
    MoeSizes sizes;
    float gain_w, gain_b;
    std::string init_method;

    MixtureOfExperts(size_t input_size, size_t hidden_size, size_t output_size, int num_experts,
                     int top_k, const std::string &activation = "relu", bool bias = true,
                     float gain_weight = 1.0f, float gain_bias = 1.0f, std::string method = "He",
                     int device_idx = 0);
    std::string get_layer_info() const override { return sizes.info(); }
    std::string get_layer_name() const override { return "MixtureOfExperts"; }
    LayerType get_layer_type() const override { return LayerType::Linear; }
    void init_weight_bias() override;
    std::unique_ptr<BaseLayer> to_cuda(int device_idx = 0) override;
};

class MixtureOfExpertsHip : public BaseLayerHip {
   public:
    MoeSizes sizes;
    float gain_w, gain_b;
    std::string init_method;

    MixtureOfExpertsHip(const MoeSizes &sizes, bool bias, float gain_weight, float gain_bias,
                        std::string method, int device_idx);
    ~MixtureOfExpertsHip() override;
    std::string get_layer_info() const override { return sizes.info(); }
    std::string get_layer_name() const override { return "MixtureOfExpertsCuda"; }
    LayerType get_layer_type() const override { return LayerType::Linear; }
    void init_weight_bias() override;
    void forward(BaseHiddenStates &input_states, BaseHiddenStates &output_states,
                 BaseTempStates &temp_states) override;
    void backward(BaseDeltaStates &input_delta_states, BaseDeltaStates &output_delta_states,
                  BaseTempStates &temp_states, bool state_udapte = true) override;
    // Expert of every choice of the last forward pass [samples][top_k], to the host.
    std::vector<int> get_expert_choices();
    void forward_replayed(int batch_size) override;

   private:
    // samples of the last forward pass, for which d_work is laid out; and what of them the
    // backward pass finds, none if that was an evaluation
    int last_batch = 0, trained_batch = 0;
    // What the last forward pass chose and computed on the way, and what the backward pass
    // computes; one allocation, as large as the largest batch seen needs.
    char *d_work = nullptr;
    size_t batch_held = 0;
    struct Work;
    Work work(int batch) const;
    void hold(int batch);
};

}  // namespace tagi_host
