// The norm of a list of gradients, and the gradients scaled to at most a given norm.
//
// The list goes to the kernels by value, as many tensors a launch as fit into 4 KB of
// arguments, cut into chunks of equal length, so tensors of any lengths fill the chip
// together.  Squares are added up in float64: a product of two floats is exact there and none
// overflows.
//
// Bound by the memory: a list larger than the caches is read twice and written once.  285
// million elements (570 MB): the norm 86 us, 6.6 TB/s (131 with plain loads), the clip 180 us,
// 6.3 TB/s; both go past the caches.  The conversions and products of float64 stay behind
// the loads.
#include "elements.hpp"
#include "operators.hpp"

namespace ilgpu_hip {

namespace {

constexpr int kBlock = 256;
constexpr int kTensors = 120;            // per launch
constexpr int kNormChunk = 32768, kClipChunk = 16384;  // bytes
constexpr int kBlocksPerCu = 8;          // of a norm: each leaves a partial sum
constexpr int64_t kMaxClipBlocks = 1 << 22;

struct TensorTable {
  const void* source[kTensors];
  void* target[kTensors];
  int64_t length[kTensors];
  uint32_t chunks_end[kTensors];         // chunks of this and all tensors before it
  int32_t type[kTensors];                // (words: a scalar load of its own each)
  int32_t count;
};
static_assert(sizeof(TensorTable) <= 4000, "kernel arguments");

// Fills `table` from tensor `next` on; returns the first tensor that is left for another
// launch.
int64_t fill_table(TensorTable& table, const ilgpu_hip_tensor* sources,
                   const ilgpu_hip_tensor* targets, int64_t count, int64_t next, int chunk) {
  int used = 0;
  int64_t chunks = 0;
  for (; next < count && used < kTensors; ++next) {
    if (sources[next].length == 0) continue;
    // (At most 2^28 and one per tensor.)
    chunks += div_up(sources[next].length * operator_elem_size(sources[next].type), chunk);
    table.source[used] = sources[next].data;
    table.target[used] = targets != nullptr ? targets[next].data : sources[next].data;
    table.length[used] = sources[next].length;
    table.chunks_end[used] = (uint32_t)chunks;
    table.type[used] = sources[next].type;
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

// Calls f(tensor, T(), first element, elements) for a chunk.
template <int CHUNK, typename F>
__device__ __forceinline__ void with_chunk(const TensorTable& table, uint32_t chunk, F f) {
  const int t = tensor_of(table, chunk);
  const int64_t in = chunk - (t > 0 ? table.chunks_end[t - 1] : 0);
  const auto call = [&](auto type) {
    constexpr int64_t kElements = CHUNK / sizeof(type);
    const int64_t left = table.length[t] - in * kElements;
    f(t, type, in * kElements, left < kElements ? left : kElements);
  };
  switch (table.type[t]) {
    case ILGPU_HIP_F32: call(float()); break;
    case ILGPU_HIP_F16: call(half_t()); break;
    default: call(bfloat_t()); break;
  }
}

// Calls f(loaded vector, its index) for the whole vectors of `count` elements, several loads
// in flight, and g(element index) for the elements that are left.
template <typename T, int U, typename F, typename G>
__device__ __forceinline__ void for_elements(const T* p, int64_t count, F f, G g) {
  constexpr int W = 16 / sizeof(T);
  using P = typename Pack<T, W>::type;
  const int vectors = (int)(count / W);
  int i = threadIdx.x;
  for (; i + (U - 1) * kBlock < vectors; i += U * kBlock) {
    typename Pack<T, W>::vec v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      v[u] = __builtin_nontemporal_load(reinterpret_cast<const P*>(p + (int64_t)(i + u * kBlock) * W));
#pragma unroll
    for (int u = 0; u < U; ++u) f(v[u], (int64_t)(i + u * kBlock) * W);
  }
  for (; i < vectors; i += kBlock) {
    const typename Pack<T, W>::vec v = *reinterpret_cast<const P*>(p + (int64_t)i * W);
    f(v, (int64_t)i * W);
  }
  const int64_t rest = (int64_t)vectors * W + threadIdx.x;
  if (rest < count) g(rest);
}

__global__ __launch_bounds__(kBlock) void square_sums_kernel(TensorTable table,
                                                             double* __restrict__ partials) {
  __shared__ double lds[kBlock / kWaveSize];
  const uint32_t chunks = table.chunks_end[table.count - 1];
  double sum = 0.0;
  for (uint32_t chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    with_chunk<kNormChunk>(table, chunk, [&](int t, auto type, int64_t from, int64_t count) {
      using T = decltype(type);
      constexpr int W = 16 / sizeof(T);
      const T* p = static_cast<const T*>(table.source[t]) + from;
      for_elements<T, kNormChunk / (16 * kBlock)>(
          p, count,
          [&](const typename Pack<T, W>::vec& v, int64_t) {
#pragma unroll
            for (int k = 0; k < W; ++k) sum += (double)(float)v[k] * (double)(float)v[k];
          },
          [&](int64_t i) { sum += (double)(float)p[i] * (double)(float)p[i]; });
    });
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

__global__ __launch_bounds__(kBlock) void clip_kernel(TensorTable table,
                                                      const float* __restrict__ norm,
                                                      float max_norm) {
  const float n = norm[0];
  // (false for NaN; an infinite norm gives no factor either)
  const bool clipped = n > max_norm && n <= 3.402823466e+38f;
  // A factor below the normal numbers has few bits: it is made 2^120 times as large, which gives
  // products of at most 2^120 max_norm, and taken back behind the product.
  const bool tiny = clipped && max_norm / n < 0x1p-126f;
  const float factor = tiny ? max_norm * 0x1p120f / n : clipped ? max_norm / n : 1.0f;
  const float back = tiny ? 0x1p-120f : 1.0f;
  const uint32_t chunks = table.chunks_end[table.count - 1];
  for (uint32_t chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    with_chunk<kClipChunk>(table, chunk, [&](int t, auto type, int64_t from, int64_t count) {
      using T = decltype(type);
      constexpr int W = 16 / sizeof(T);
      if (!clipped && table.source[t] == table.target[t]) return;
      const T* source = static_cast<const T*>(table.source[t]) + from;
      T* target = static_cast<T*>(table.target[t]) + from;  // perhaps the source
      for_elements<T, kClipChunk / (16 * kBlock)>(
          source, count,
          [&](const typename Pack<T, W>::vec& v, int64_t at) {
            typename Pack<T, W>::vec r;
#pragma unroll
            for (int k = 0; k < W; ++k) r[k] = (T)product_for<T>((float)v[k] * factor, back);
            __builtin_nontemporal_store(r, reinterpret_cast<typename Pack<T, W>::type*>(target + at));
          },
          [&](int64_t at) { target[at] = (T)product_for<T>((float)source[at] * factor, back); });
    });
  }
}

inline int64_t max_blocks() { return (int64_t)device_cu_count() * kBlocksPerCu; }
inline int64_t blocks_for(const TensorTable& table) {
  const int64_t chunks = table.chunks_end[table.count - 1];
  return chunks < max_blocks() ? chunks : max_blocks();
}

// A block for every chunk of a clip (285 million elements, norm and clip, us: 270; eight blocks
// a compute unit that take chunks in turn 285, with chunks of 32 KB 288, of 8 KB 271).
inline int64_t clip_blocks(const TensorTable& table) {
  const int64_t chunks = table.chunks_end[table.count - 1];
  return chunks < kMaxClipBlocks ? chunks : kMaxClipBlocks;
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
    next = fill_table(table, tensors, nullptr, count, next, kNormChunk);
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
    next = fill_table(table, sources, targets, count, next, kClipChunk);
    if (table.count == 0) break;
    {
      ProfileScope scope(stream, "clip_gradients");
      hipLaunchKernelGGL(clip_kernel, dim3((unsigned)clip_blocks(table)), dim3(kBlock), 0, stream,
                         table, norm, max_norm);
    }
    ILGPU_HIP_CHECK(hipGetLastError());
  }
  return ILGPU_HIP_SUCCESS;
}

}  // namespace ilgpu_hip
