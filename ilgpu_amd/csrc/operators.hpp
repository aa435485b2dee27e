// Launch entry points of the operators of language models.
#pragma once

#include "kernels.hpp"

namespace ilgpu_hip {

// embedding.hip.  `count` may be 0; float32 scale; types and strides as the C ABI has them.
struct EmbeddingArgs {
  const void* table;
  int64_t vocabulary, dimension, table_stride;
  int32_t table_type;
  const void* tokens;
  int64_t count;
  int32_t token_type;
  float scale;
  void* out;
  int64_t out_stride;
  int32_t out_type;
};
int32_t launch_embedding(hipStream_t stream, const EmbeddingArgs& args);
struct EmbeddingGradientArgs {
  const void* grad_out;
  int64_t grad_out_stride;
  int32_t grad_out_type;
  const void* tokens;
  int64_t count;
  int32_t token_type;
  float scale;
  int64_t padding_token;
  int32_t accumulate;
  void* grad_table;
  int64_t vocabulary, dimension, table_stride;
  int32_t table_type;
  void* temp;
};
int64_t embedding_gradient_temp_bytes(int64_t count, int64_t vocabulary, int64_t dimension);
int32_t launch_embedding_gradient(hipStream_t stream, const EmbeddingGradientArgs& args);

// layer_norm.hip.  `rows` may be 0.
struct LayerNormArgs {
  const void* in;
  int64_t rows, columns, in_stride;
  int32_t type;
  const void* weight;  // weight, bias, mean and rstd may be nullptr
  const void* bias;
  int32_t weight_type;
  float epsilon;
  void* out;
  int64_t out_stride;
  float* mean;
  float* rstd;
};
int32_t launch_layer_norm(hipStream_t stream, const LayerNormArgs& args);
struct LayerNormGradientArgs {
  const void* grad_out;
  int64_t grad_out_stride;
  const void* in;
  int64_t in_stride, rows, columns;
  int32_t type;
  const void* weight;  // may be nullptr
  int32_t weight_type;
  const float* mean;
  const float* rstd;
  void* grad_in;       // each may be nullptr
  int64_t grad_in_stride;
  void* grad_weight;
  void* grad_bias;
  int32_t accumulate;
  void* temp;
};
int64_t layer_norm_gradient_temp_bytes(int64_t rows, int64_t columns);
int32_t launch_layer_norm_gradient(hipStream_t stream, const LayerNormGradientArgs& args);

// gradient_norm.hip
int64_t gradient_norm_temp_bytes(int64_t count);
int32_t launch_gradient_norm(hipStream_t stream, const ilgpu_hip_tensor* tensors, int64_t count,
                             float* norm, void* temp);
int32_t launch_clip_gradients(hipStream_t stream, const ilgpu_hip_tensor* sources,
                              const ilgpu_hip_tensor* targets, int64_t count, const float* norm,
                              float max_norm);

// gated_recurrence.hip.  `rows` may be 0.
struct GatedRecurrenceArgs {
  const void* gate;
  int64_t gate_stride;
  const void* in;
  int64_t in_stride, rows, channels;
  int32_t type, decay, complement;
  const void* offsets;  // nullptr: equal parts
  int32_t offset_type;
  int64_t sequences;
  const float* initial;  // may be nullptr
  int64_t initial_stride;
  void* out;             // backwards: as the forward call left it
  int64_t out_stride;
  float* final_state;    // may be nullptr
  int64_t final_stride;
  bool backwards;
  const void* grad_out;
  int64_t grad_out_stride;
  const float* grad_final;  // may be nullptr
  int64_t grad_final_stride;
  void* grad_gate;       // each may be nullptr
  int64_t grad_gate_stride;
  void* grad_in;
  int64_t grad_in_stride;
  float* grad_initial;
  int64_t grad_initial_stride;
  void* temp;
};
int64_t gated_recurrence_temp_bytes(int64_t rows, int64_t channels);
int32_t launch_gated_recurrence(hipStream_t stream, const GatedRecurrenceArgs& args);

// residual_norm.hip.  `rows` may be 0; what is said to be optional in the C ABI may be nullptr.
struct ResidualNormArgs {
  const void* in;
  int64_t in_stride, rows, columns;
  int32_t type, input_norm;
  const void* input_weight;
  const void* gate;
  int64_t gate_stride;
  int32_t gate_kind;
  const void* residual;
  int64_t residual_stride;
  int32_t residual_type;
  float scale;
  const void* weight;
  int32_t weight_type;
  float epsilon;
  void* total;
  int64_t total_stride;
  void* out;
  int64_t out_stride;
  float* input_rstd;
  float* rstd;
};
int32_t launch_residual_norm(hipStream_t stream, const ResidualNormArgs& args);
struct ResidualNormGradientArgs {
  const void* grad_out;
  int64_t grad_out_stride;
  const void* grad_total;
  int64_t grad_total_stride;
  const void* in;
  int64_t in_stride, rows, columns;
  int32_t type, input_norm;
  const void* input_weight;
  const float* input_rstd;
  const void* gate;
  int64_t gate_stride;
  int32_t gate_kind;
  const void* total;
  int64_t total_stride;
  int32_t residual_type;
  float scale;
  const void* weight;
  int32_t weight_type;
  const float* rstd;
  void* grad_in;
  int64_t grad_in_stride;
  void* grad_gate;
  int64_t grad_gate_stride;
  void* grad_residual;
  int64_t grad_residual_stride;
  void* grad_input_weight;
  void* grad_weight;
  int32_t accumulate;
};
int64_t residual_norm_gradient_temp_bytes(int64_t rows, int64_t columns);
int32_t launch_residual_norm_gradient(hipStream_t stream, const ResidualNormGradientArgs& args,
                                      void* temp);

// adamw.hip.  Scales nullptr: moments in 32 bits; copies, schedule and norm may be nullptr.
struct AdamwArgs {
  const ilgpu_hip_tensor* parameters;
  const ilgpu_hip_tensor* gradients;
  const ilgpu_hip_tensor* first;
  const ilgpu_hip_tensor* second;
  const ilgpu_hip_tensor* first_scales;
  const ilgpu_hip_tensor* second_scales;
  const ilgpu_hip_tensor* copies;
  int64_t count;
  ilgpu_hip_adamw_options options;
  const int64_t* step;
  const float* schedule;
  const float* norm;
};
constexpr int kMomentBlock = 256;  // moments in 8 bits that share a scale
int32_t launch_adamw(hipStream_t stream, const AdamwArgs& args);
int32_t launch_adamw_moments(hipStream_t stream, const ilgpu_hip_tensor* codes,
                             const ilgpu_hip_tensor* scales, const ilgpu_hip_tensor* targets,
                             int64_t count, bool second);

}  // namespace ilgpu_hip
