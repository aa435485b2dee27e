// The norm of a list of gradients, and the gradients scaled to at most a given norm.
//
// The list goes to the kernels by value, as many tensors a launch as fit into 4 KB of
// arguments, cut into chunks of equal length; blocks take chunks in turn, so tensors
// of any lengths fill the chip together.  Squares are added up in float64: a product
// of two floats is exact there and none overflows.
#include "elements.hpp"
#include "kernels.hpp"

namespace ilgpu_hip {

namespace {

constexpr int kBlock = 256;
constexpr int kTensors = 128;            // per launch
constexpr int64_t kChunk = 16384;        // elements
constexpr int kBlocksPerCu = 8;

struct TensorTable {
  const void* source[kTensors];
  void* target[kTensors];
  int64_t length[kTensors];
  uint32_t chunks_end[kTensors];         // chunks of this and all tensors before it
  uint8_t type[kTensors];
  int32_t count;
};
static_assert(sizeof(TensorTable) <= 4000, "kernel arguments");

// Fills `table` from tensor `next` on; returns the first tensor that is left for another
// launch.
int64_t fill_table(TensorTable& table, const ilgpu_hip_tensor* sources,
                   const ilgpu_hip_tensor* targets, int64_t count, int64_t next) {
  int used = 0;
  int64_t chunks = 0;
  for (; next < count && used < kTensors; ++next) {
    if (sources[next].length == 0) continue;
    chunks += div_up(sources[next].length, kChunk);  // at most 2^26 and one per tensor
    table.source[used] = sources[next].data;
    table.target[used] = targets != nullptr ? targets[next].data : sources[next].data;
    table.length[used] = sources[next].length;
    table.chunks_end[used] = (uint32_t)chunks;
    table.type[used] = (uint8_t)sources[next].type;
    ++used;
  }
  table.count = used;
  return next;
}

__device__ __forceinline__ int tensor_of(const TensorTable& table, uint32_t chunk) {
  int low = 0, high = table.count - 1;
  while (low < high) {
    const int middle = (low + high) >> 1;
    if (table.chunks_end[middle] <= chunk) low = middle + 1;
    else high = middle;
  }
  return low;
}

__device__ __forceinline__ double block_sum(double v, double* lds) {
#pragma unroll
  for (int off = kWaveSize / 2; off > 0; off >>= 1) v += shfl_down(v, off);
  if ((threadIdx.x & (kWaveSize - 1)) == 0) lds[threadIdx.x / kWaveSize] = v;
  __syncthreads();
  double sum = 0.0;
#pragma unroll
  for (int w = 0; w < kBlock / kWaveSize; ++w) sum += lds[w];
  return sum;
}

template <typename T>
__device__ __forceinline__ double chunk_squares(const T* p, int64_t count) {
  constexpr int W = 16 / sizeof(T);
  double sum = 0.0;
  for (int64_t i = (int64_t)threadIdx.x * W; i < count; i += kBlock * W) {
    float v[W];
    load_floats<T, W>(v, p + i, count - i);
#pragma unroll
    for (int k = 0; k < W; ++k) sum += (double)v[k] * (double)v[k];
  }
  return sum;
}

__global__ __launch_bounds__(kBlock) void square_sums_kernel(TensorTable table,
                                                             double* __restrict__ partials) {
  __shared__ double lds[kBlock / kWaveSize];
  const uint32_t chunks = table.chunks_end[table.count - 1];
  double sum = 0.0;
  for (uint32_t chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    const int t = tensor_of(table, chunk);
    const int64_t from = (int64_t)(chunk - (t > 0 ? table.chunks_end[t - 1] : 0)) * kChunk;
    const int64_t left = table.length[t] - from;
    const int64_t count = left < kChunk ? left : kChunk;
    switch (table.type[t]) {
      case ILGPU_HIP_F32:
        sum += chunk_squares(static_cast<const float*>(table.source[t]) + from, count);
        break;
      case ILGPU_HIP_F16:
        sum += chunk_squares(static_cast<const half_t*>(table.source[t]) + from, count);
        break;
      default:
        sum += chunk_squares(static_cast<const bfloat_t*>(table.source[t]) + from, count);
        break;
    }
  }
  sum = block_sum(sum, lds);
  if (threadIdx.x == 0) partials[blockIdx.x] = sum;
}

__global__ __launch_bounds__(kBlock) void norm_kernel(const double* __restrict__ partials,
                                                      int64_t count, float* __restrict__ norm) {
  __shared__ double lds[kBlock / kWaveSize];
  double sum = 0.0;
  for (int64_t i = threadIdx.x; i < count; i += kBlock) sum += partials[i];
  sum = block_sum(sum, lds);
  if (threadIdx.x == 0) norm[0] = (float)sqrt(sum);
}

// source and target may be the same array.
template <typename T>
__device__ __forceinline__ void scale_chunk(const T* source, T* target, int64_t count,
                                            float factor) {
  constexpr int W = 16 / sizeof(T);
  for (int64_t i = (int64_t)threadIdx.x * W; i < count; i += kBlock * W) {
    float v[W];
    load_floats<T, W>(v, source + i, count - i);
#pragma unroll
    for (int k = 0; k < W; ++k) v[k] *= factor;
    store_floats<T, W>(target + i, v, count - i);
  }
}

__global__ __launch_bounds__(kBlock) void clip_kernel(TensorTable table,
                                                      const float* __restrict__ norm,
                                                      float max_norm) {
  const float n = norm[0];
  // (false for NaN; an infinite norm gives no factor either)
  const bool clipped = n > max_norm && n <= 3.402823466e+38f;
  const float factor = clipped ? max_norm / n : 1.0f;
  const uint32_t chunks = table.chunks_end[table.count - 1];
  for (uint32_t chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    const int t = tensor_of(table, chunk);
    if (!clipped && table.source[t] == table.target[t]) continue;
    const int64_t from = (int64_t)(chunk - (t > 0 ? table.chunks_end[t - 1] : 0)) * kChunk;
    const int64_t left = table.length[t] - from;
    const int64_t count = left < kChunk ? left : kChunk;
    switch (table.type[t]) {
      case ILGPU_HIP_F32:
        scale_chunk(static_cast<const float*>(table.source[t]) + from,
                    static_cast<float*>(table.target[t]) + from, count, factor);
        break;
      case ILGPU_HIP_F16:
        scale_chunk(static_cast<const half_t*>(table.source[t]) + from,
                    static_cast<half_t*>(table.target[t]) + from, count, factor);
        break;
      default:
        scale_chunk(static_cast<const bfloat_t*>(table.source[t]) + from,
                    static_cast<bfloat_t*>(table.target[t]) + from, count, factor);
        break;
    }
  }
}

inline int64_t max_blocks() { return (int64_t)device_cu_count() * kBlocksPerCu; }
inline int64_t blocks_for(const TensorTable& table) {
  const int64_t chunks = table.chunks_end[table.count - 1];
  return chunks < max_blocks() ? chunks : max_blocks();
}

}  // namespace

// Partial sums of every launch: one for each kTensors tensors begun.
int64_t gradient_norm_temp_bytes(int64_t count) {
  return (div_up(count, kTensors) + 1) * max_blocks() * 8 + 16;
}

int32_t launch_gradient_norm(hipStream_t stream, const ilgpu_hip_tensor* tensors, int64_t count,
                             float* norm, void* temp) {
  double* partials = reinterpret_cast<double*>(align_up((int64_t)(uintptr_t)temp, 16));
  int64_t used = 0;
  TensorTable table;
  for (int64_t next = 0; next < count;) {
    next = fill_table(table, tensors, nullptr, count, next);
    if (table.count == 0) break;
    const int64_t blocks = blocks_for(table);
    {
      ProfileScope scope(stream, "gradient_square_sums");
      hipLaunchKernelGGL(square_sums_kernel, dim3((unsigned)blocks), dim3(kBlock), 0, stream,
                         table, partials + used);
    }
    ILGPU_HIP_CHECK(hipGetLastError());
    used += blocks;
  }
  {
    ProfileScope scope(stream, "gradient_norm");
    hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(kBlock), 0, stream, partials, used, norm);
  }
  ILGPU_HIP_CHECK(hipGetLastError());
  return ILGPU_HIP_SUCCESS;
}

int32_t launch_clip_gradients(hipStream_t stream, const ilgpu_hip_tensor* sources,
                              const ilgpu_hip_tensor* targets, int64_t count, const float* norm,
                              float max_norm) {
  TensorTable table;
  for (int64_t next = 0; next < count;) {
    next = fill_table(table, sources, targets, count, next);
    if (table.count == 0) break;
    {
      ProfileScope scope(stream, "clip_gradients");
      hipLaunchKernelGGL(clip_kernel, dim3((unsigned)blocks_for(table)), dim3(kBlock), 0, stream,
                         table, norm, max_norm);
    }
    ILGPU_HIP_CHECK(hipGetLastError());
  }
  return ILGPU_HIP_SUCCESS;
}

}  // namespace ilgpu_hip
