// Embedding lookup, out[i] = scale * table[tokens[i]], and its gradient,
// grad_table[v] = scale * sum of grad_out[i] over the positions of token v.
#include "elements.hpp"
#include "kernels.hpp"

namespace ilgpu_hip {

namespace {

constexpr int kBlock = 256;
constexpr int64_t kMaxBlocks = 1 << 22;  // blocks go on to further rows beyond

// Lanes that share a row: a power of two, at most a block.
inline int lanes_log2(int64_t dimension, int width) {
  int log2 = 0;
  while ((1 << log2) < kBlock && ((int64_t)width << log2) < dimension) ++log2;
  return log2;
}
inline unsigned row_blocks(int64_t rows, int log2) {
  const int64_t blocks = div_up(rows, kBlock >> log2);
  return (unsigned)(blocks < kMaxBlocks ? blocks : kMaxBlocks);
}

template <typename TI, typename TO> struct Width {
  static constexpr int value = 16 / (sizeof(TI) > sizeof(TO) ? sizeof(TI) : sizeof(TO));
};

template <typename TI, typename TO, typename TT>
__global__ __launch_bounds__(kBlock) void embedding_kernel(
    const TI* __restrict__ table, int64_t vocabulary, int64_t dimension, int64_t table_stride,
    const TT* __restrict__ tokens, int64_t count, float scale, TO* __restrict__ out,
    int64_t out_stride, int log2) {
  constexpr int W = Width<TI, TO>::value;
  const int64_t rows_per_block = kBlock >> log2;
  const int64_t first = (int64_t)(threadIdx.x & ((1u << log2) - 1)) * W;
  for (int64_t i = blockIdx.x * rows_per_block + (threadIdx.x >> log2); i < count;
       i += gridDim.x * rows_per_block) {
    const int64_t token = (int64_t)tokens[i];
    const bool there = (uint64_t)token < (uint64_t)vocabulary;
    const TI* from = table + (there ? token : 0) * table_stride;
    TO* to = out + i * out_stride;
    for (int64_t c = first; c < dimension; c += (int64_t)W << log2) {
      float v[W];
      load_floats<TI, W>(v, from + c, there ? dimension - c : 0);
#pragma unroll
      for (int k = 0; k < W; ++k) v[k] = there ? v[k] * scale : 0.0f;
      store_floats<TO, W>(to + c, v, dimension - c);
    }
  }
}

// Sort keys of the positions: their tokens, `vocabulary` for those that count nowhere.
template <typename TT>
__global__ __launch_bounds__(kBlock) void token_keys_kernel(
    const TT* __restrict__ tokens, int64_t count, int64_t vocabulary, int64_t padding_token,
    uint32_t* __restrict__ keys) {
  for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < count;
       i += (int64_t)gridDim.x * kBlock) {
    const int64_t token = (int64_t)tokens[i];
    const bool counts = (uint64_t)token < (uint64_t)vocabulary && token != padding_token;
    keys[i] = (uint32_t)(counts ? token : vocabulary);
  }
}

// Each row of the table finds its positions in the sorted keys and adds them up in
// the order of the positions.
template <typename TG, typename TW>
__global__ __launch_bounds__(kBlock) void embedding_gradient_kernel(
    const TG* __restrict__ grad_out, int64_t grad_out_stride, const uint32_t* __restrict__ keys,
    const uint32_t* __restrict__ order, int64_t count, float scale, int32_t accumulate,
    TW* __restrict__ grad_table, int64_t vocabulary, int64_t dimension, int64_t table_stride,
    int log2) {
  constexpr int W = Width<TG, TW>::value;
  const int64_t rows_per_block = kBlock >> log2;
  const int64_t first = (int64_t)(threadIdx.x & ((1u << log2) - 1)) * W;
  for (int64_t row = blockIdx.x * rows_per_block + (threadIdx.x >> log2); row < vocabulary;
       row += gridDim.x * rows_per_block) {
    int64_t low = 0, high = count;
    while (low < high) {
      const int64_t middle = (low + high) >> 1;
      if ((int64_t)keys[middle] < row) low = middle + 1;
      else high = middle;
    }
    const bool met = low < count && (int64_t)keys[low] == row;
    if (!met && accumulate) continue;
    TW* to = grad_table + row * table_stride;
    for (int64_t c = first; c < dimension; c += (int64_t)W << log2) {
      float sum[W];
#pragma unroll
      for (int k = 0; k < W; ++k) sum[k] = 0.0f;
      for (int64_t p = low; p < count && (int64_t)keys[p] == row; ++p) {
        float v[W];
        load_floats<TG, W>(v, grad_out + (int64_t)order[p] * grad_out_stride + c, dimension - c);
#pragma unroll
        for (int k = 0; k < W; ++k) sum[k] += v[k];
      }
      float old[W];
      load_floats<TW, W>(old, to + c, accumulate ? dimension - c : 0);
#pragma unroll
      for (int k = 0; k < W; ++k) sum[k] = sum[k] * scale + old[k];
      store_floats<TW, W>(to + c, sum, dimension - c);
    }
  }
}

struct GradientTemp {
  int64_t keys, order, sort, bytes;  // offsets
};
GradientTemp gradient_temp(int64_t count) {
  GradientTemp t;
  t.keys = 0;
  t.order = align_up(count * 4, 256);
  t.sort = 2 * t.order;
  t.bytes = t.sort + (count > 0 ? radix_sort_temp_bytes(count, 4, 4) : 0) + 256;
  return t;
}

}  // namespace

int32_t launch_embedding(hipStream_t stream, const EmbeddingArgs& a) {
  if (a.count == 0) return ILGPU_HIP_SUCCESS;
  return with_type(a.table_type, [&](auto ti) {
    return with_type(a.out_type, [&](auto to) {
      return with_token_type(a.token_type, [&](auto tt) -> int32_t {
        using TI = decltype(ti);
        using TO = decltype(to);
        using TT = decltype(tt);
        const int log2 = lanes_log2(a.dimension, Width<TI, TO>::value);
        {
          ProfileScope scope(stream, "embedding");
          hipLaunchKernelGGL((embedding_kernel<TI, TO, TT>), dim3(row_blocks(a.count, log2)),
                             dim3(kBlock), 0, stream, static_cast<const TI*>(a.table),
                             a.vocabulary, a.dimension, a.table_stride,
                             static_cast<const TT*>(a.tokens), a.count, a.scale,
                             static_cast<TO*>(a.out), a.out_stride, log2);
        }
        ILGPU_HIP_CHECK(hipGetLastError());
        return ILGPU_HIP_SUCCESS;
      });
    });
  });
}

int64_t embedding_gradient_temp_bytes(int64_t count, int64_t, int64_t) {
  return gradient_temp(count).bytes;
}

int32_t launch_embedding_gradient(hipStream_t stream, const EmbeddingGradientArgs& a) {
  if (a.vocabulary == 0) return ILGPU_HIP_SUCCESS;
  if (a.count > 0) {
    const int32_t rc = check_sort_device(stream);  // before anything is launched
    if (rc != ILGPU_HIP_SUCCESS) return rc;
  }
  const GradientTemp t = gradient_temp(a.count);
  char* base = reinterpret_cast<char*>(align_up((int64_t)(uintptr_t)a.temp, 256));
  uint32_t* keys = reinterpret_cast<uint32_t*>(base + t.keys);
  uint32_t* order = reinterpret_cast<uint32_t*>(base + t.order);
  if (a.count > 0) {
    const int32_t rc = with_token_type(a.token_type, [&](auto tt) -> int32_t {
      using TT = decltype(tt);
      const int64_t blocks = div_up(a.count, kBlock);
      ProfileScope scope(stream, "embedding_token_keys");
      hipLaunchKernelGGL((token_keys_kernel<TT>),
                         dim3((unsigned)(blocks < kMaxBlocks ? blocks : kMaxBlocks)),
                         dim3(kBlock), 0, stream, static_cast<const TT*>(a.tokens), a.count,
                         a.vocabulary, a.padding_token, keys);
      ILGPU_HIP_CHECK(hipGetLastError());
      return ILGPU_HIP_SUCCESS;
    });
    if (rc != ILGPU_HIP_SUCCESS) return rc;
    const SortArgs sort{keys, order, 1, 1, a.count, ILGPU_HIP_U32, 4, 0,
                        ILGPU_HIP_VALUES_FROM_INDEX, base + t.sort};
    const int32_t sorted = launch_radix_sort(stream, sort);
    if (sorted != ILGPU_HIP_SUCCESS) return sorted;
  }
  return with_type(a.grad_out_type, [&](auto tg) {
    return with_type(a.table_type, [&](auto tw) -> int32_t {
      using TG = decltype(tg);
      using TW = decltype(tw);
      const int log2 = lanes_log2(a.dimension, Width<TG, TW>::value);
      {
        ProfileScope scope(stream, "embedding_gradient");
        hipLaunchKernelGGL((embedding_gradient_kernel<TG, TW>),
                           dim3(row_blocks(a.vocabulary, log2)), dim3(kBlock), 0, stream,
                           static_cast<const TG*>(a.grad_out), a.grad_out_stride, keys, order,
                           a.count, a.scale, a.accumulate, static_cast<TW*>(a.grad_table),
                           a.vocabulary, a.dimension, a.table_stride, log2);
      }
      ILGPU_HIP_CHECK(hipGetLastError());
      return ILGPU_HIP_SUCCESS;
    });
  });
}

}  // namespace ilgpu_hip
