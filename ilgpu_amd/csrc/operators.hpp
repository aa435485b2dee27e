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

}  // namespace ilgpu_hip
