// Layer norm of the rows of a matrix, and its gradients.
//
// Sums are in float32, of a thread's own elements first and then over the block
// in a fixed order; the variance is the mean of the squared deviations from the
// mean already known, which loses nothing where the mean is large against them.
#include "elements.hpp"
#include "kernels.hpp"

namespace ilgpu_hip {

namespace {

constexpr int kBlock = 256;
constexpr int64_t kMaxBlocks = 1 << 22;
constexpr int kMaxSplits = 256;

__device__ __forceinline__ float block_sum(float v, float* lds) {
#pragma unroll
  for (int off = kWaveSize / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, kWaveSize);
  __syncthreads();
  if ((threadIdx.x & (kWaveSize - 1)) == 0) lds[threadIdx.x / kWaveSize] = v;
  __syncthreads();
  float sum = 0.0f;
#pragma unroll
  for (int w = 0; w < kBlock / kWaveSize; ++w) sum += lds[w];
  return sum;
}

template <typename T, typename TW>
__global__ __launch_bounds__(kBlock) void layer_norm_kernel(
    const T* in, int64_t rows, int64_t columns, int64_t in_stride, const TW* __restrict__ weight,
    const TW* __restrict__ bias, float epsilon, T* out, int64_t out_stride,
    float* __restrict__ mean, float* __restrict__ rstd) {
  __shared__ float lds[kBlock / kWaveSize];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* x = in + row * in_stride;
    float sum = 0.0f;
    for (int64_t c = threadIdx.x; c < columns; c += kBlock) sum += (float)x[c];
    const float m = block_sum(sum, lds) / (float)columns;
    sum = 0.0f;
    for (int64_t c = threadIdx.x; c < columns; c += kBlock) {
      const float d = (float)x[c] - m;
      sum += d * d;
    }
    const float r = 1.0f / sqrtf(block_sum(sum, lds) / (float)columns + epsilon);
    T* y = out + row * out_stride;
    for (int64_t c = threadIdx.x; c < columns; c += kBlock) {
      const float w = weight != nullptr ? (float)weight[c] : 1.0f;
      const float b = bias != nullptr ? (float)bias[c] : 0.0f;
      y[c] = (T)(((float)x[c] - m) * r * w + b);
    }
    if (threadIdx.x == 0) {
      if (mean != nullptr) mean[row] = m;
      if (rstd != nullptr) rstd[row] = r;
    }
  }
}

template <typename T, typename TW>
__global__ __launch_bounds__(kBlock) void layer_norm_grad_in_kernel(
    const T* grad_out, int64_t grad_out_stride, const T* in, int64_t in_stride, int64_t rows,
    int64_t columns, const TW* __restrict__ weight, const float* __restrict__ mean,
    const float* __restrict__ rstd, T* grad_in, int64_t grad_in_stride) {
  __shared__ float lds[kBlock / kWaveSize];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* x = in + row * in_stride;
    const T* dy = grad_out + row * grad_out_stride;
    const float m = mean[row], r = rstd[row];
    float sum_g = 0.0f, sum_gh = 0.0f;
    for (int64_t c = threadIdx.x; c < columns; c += kBlock) {
      const float g = (float)dy[c] * (weight != nullptr ? (float)weight[c] : 1.0f);
      sum_g += g;
      sum_gh += g * (((float)x[c] - m) * r);
    }
    const float mean_g = block_sum(sum_g, lds) / (float)columns;
    const float mean_gh = block_sum(sum_gh, lds) / (float)columns;
    T* dx = grad_in + row * grad_in_stride;
    for (int64_t c = threadIdx.x; c < columns; c += kBlock) {
      const float g = (float)dy[c] * (weight != nullptr ? (float)weight[c] : 1.0f);
      const float h = ((float)x[c] - m) * r;
      dx[c] = (T)(r * (g - mean_g - h * mean_gh));
    }
  }
}

// Block (x, y): columns [256 x, 256 x + 256) over every gridDim.y-th row from y on.
// partials: gridDim.y rows of `columns` sums for the weight, then as many for the bias.
template <typename T>
__global__ __launch_bounds__(kBlock) void layer_norm_column_sums_kernel(
    const T* __restrict__ grad_out, int64_t grad_out_stride, const T* __restrict__ in,
    int64_t in_stride, int64_t rows, int64_t columns, const float* __restrict__ mean,
    const float* __restrict__ rstd, float* __restrict__ partials) {
  const int64_t c = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  if (c >= columns) return;
  float sum_w = 0.0f, sum_b = 0.0f;
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    const float dy = (float)grad_out[row * grad_out_stride + c];
    sum_w += dy * (((float)in[row * in_stride + c] - mean[row]) * rstd[row]);
    sum_b += dy;
  }
  partials[blockIdx.y * columns + c] = sum_w;
  partials[((int64_t)gridDim.y + blockIdx.y) * columns + c] = sum_b;
}

template <typename TW>
__global__ __launch_bounds__(kBlock) void layer_norm_fold_kernel(
    const float* __restrict__ partials, int64_t splits, int64_t columns, int32_t accumulate,
    TW* __restrict__ grad_weight, TW* __restrict__ grad_bias) {
  const int64_t c = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  TW* to = blockIdx.y == 0 ? grad_weight : grad_bias;
  if (c >= columns || to == nullptr) return;
  float sum = 0.0f;
  for (int64_t s = 0; s < splits; ++s) sum += partials[(blockIdx.y * splits + s) * columns + c];
  to[c] = (TW)(accumulate ? (float)to[c] + sum : sum);
}

inline int64_t column_splits(int64_t rows) { return rows < kMaxSplits ? rows : kMaxSplits; }
inline unsigned row_grid(int64_t rows) { return (unsigned)(rows < kMaxBlocks ? rows : kMaxBlocks); }

}  // namespace

int32_t launch_layer_norm(hipStream_t stream, const LayerNormArgs& a) {
  if (a.rows == 0) return ILGPU_HIP_SUCCESS;
  return with_type(a.type, [&](auto t) {
    return with_type(a.weight_type, [&](auto tw) -> int32_t {
      using T = decltype(t);
      using TW = decltype(tw);
      {
        ProfileScope scope(stream, "layer_norm");
        hipLaunchKernelGGL((layer_norm_kernel<T, TW>), dim3(row_grid(a.rows)), dim3(kBlock), 0,
                           stream, static_cast<const T*>(a.in), a.rows, a.columns, a.in_stride,
                           static_cast<const TW*>(a.weight), static_cast<const TW*>(a.bias),
                           a.epsilon, static_cast<T*>(a.out), a.out_stride, a.mean, a.rstd);
      }
      ILGPU_HIP_CHECK(hipGetLastError());
      return ILGPU_HIP_SUCCESS;
    });
  });
}

int64_t layer_norm_gradient_temp_bytes(int64_t rows, int64_t columns) {
  return 2 * column_splits(rows) * columns * 4 + 16;
}

int32_t launch_layer_norm_gradient(hipStream_t stream, const LayerNormGradientArgs& a) {
  float* partials = reinterpret_cast<float*>(align_up((int64_t)(uintptr_t)a.temp, 16));
  return with_type(a.type, [&](auto t) {
    return with_type(a.weight_type, [&](auto tw) -> int32_t {
      using T = decltype(t);
      using TW = decltype(tw);
      const unsigned column_blocks = (unsigned)div_up(a.columns, kBlock);
      // The column sums come first: grad_in may be written over what they read.
      if (a.grad_weight != nullptr || a.grad_bias != nullptr) {
        const int64_t splits = column_splits(a.rows);
        if (splits > 0) {
          ProfileScope scope(stream, "layer_norm_column_sums");
          hipLaunchKernelGGL((layer_norm_column_sums_kernel<T>),
                             dim3(column_blocks, (unsigned)splits), dim3(kBlock), 0, stream,
                             static_cast<const T*>(a.grad_out), a.grad_out_stride,
                             static_cast<const T*>(a.in), a.in_stride, a.rows, a.columns, a.mean,
                             a.rstd, partials);
        }
        ILGPU_HIP_CHECK(hipGetLastError());
        {
          ProfileScope scope(stream, "layer_norm_fold");
          hipLaunchKernelGGL((layer_norm_fold_kernel<TW>), dim3(column_blocks, 2), dim3(kBlock),
                             0, stream, partials, splits, a.columns, a.accumulate,
                             static_cast<TW*>(a.grad_weight), static_cast<TW*>(a.grad_bias));
        }
        ILGPU_HIP_CHECK(hipGetLastError());
      }
      if (a.grad_in != nullptr && a.rows > 0) {
        {
          ProfileScope scope(stream, "layer_norm_grad_in");
          hipLaunchKernelGGL((layer_norm_grad_in_kernel<T, TW>), dim3(row_grid(a.rows)),
                             dim3(kBlock), 0, stream, static_cast<const T*>(a.grad_out),
                             a.grad_out_stride, static_cast<const T*>(a.in), a.in_stride, a.rows,
                             a.columns, static_cast<const TW*>(a.weight), a.mean, a.rstd,
                             static_cast<T*>(a.grad_in), a.grad_in_stride);
        }
        ILGPU_HIP_CHECK(hipGetLastError());
      }
      return ILGPU_HIP_SUCCESS;
    });
  });
}

}  // namespace ilgpu_hip
