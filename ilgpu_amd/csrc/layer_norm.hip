// Layer norm of the rows of a matrix, and its gradients.
//
// Sums are in float32, of a thread's own elements first and then over the lanes and
// waves in a fixed order; the variance is the mean of the squared deviations from the
// mean already known.  That mean is off by some roundings of the row's size: of a row far from
// zero (far_from_zero) the deviations themselves, which are small, are added up too, and
// mean, deviations and variance are put right by their mean.
//
// Bound by the memory: a row is read once, stays in the registers of the wave or block
// that normalises it, and is written once.  Waves and blocks go from row to row and hold
// the weights of their columns; the next row is on its way while one is worked on.  32768 x
// 4096 bfloat16: 537 MB in 98 us, 5.5 TB/s (three readings from the caches, element by
// element: 338).
#include "operators.hpp"
#include "rows.hpp"

namespace ilgpu_hip {

namespace {

// Whether a row's mean is more than two deviations from zero. Below that its roundings are as
// small as those of the deviations' own sums; beyond it a third sum finds the `rest` of the
// mean: 32768 x 4096 bfloat16 100 us where all rows are far, 98 where none is.  (Added up in every
// row: 8192 x 2000 bfloat16 15.2 instead of 13.6, 4099 x 1537 float16 9.5 instead of 8.9.)
template <int LANES> __device__ __forceinline__ bool far_from_zero(float mean, float variance) {
  const int far = mean * mean > 4.0f * variance;
  return __builtin_expect(LANES >= kWaveSize ? __builtin_amdgcn_readfirstlane(far) : far, 0);
}
__device__ __forceinline__ float less_rest(float variance, float rest) {
  return fmaxf(variance - rest * rest, 0.0f);
}

// Blocks of a launch, in waves a compute unit: twice as many as are resident, so that the
// last rows are spread (32768 x 4096, us: 104.6 with 32, 99.9 with 64, 99.7 with 128, 124
// with a block for every row, which loads its weights for it alone; that is what a few thousand
// rows get).
constexpr int kWavesPerCu = 64;

// Rows of more vectors have two in a thread (32768 x 4096: 512 vectors by 256 threads 98 us, by
// 512 101.7).
constexpr int kSingleVectors = 384;

template <typename T, typename TW, int W, int LANES, int V>
__global__ __launch_bounds__(row_block<LANES>()) void layer_norm_kernel(
    const T* in, int64_t rows, int64_t columns, int64_t in_stride, const TW* __restrict__ weight,
    const TW* __restrict__ bias, float epsilon, T* out, int64_t out_stride,
    float* __restrict__ mean, float* __restrict__ rstd) {
  constexpr int kRows = block_rows<LANES>();
  __shared__ float lds[3][kMostWaves];
  const Columns<W, LANES, V> own(columns);
  const int64_t step = (int64_t)gridDim.x * kRows;
  int64_t row = (int64_t)blockIdx.x * kRows + row_of_block<LANES>();
  if (row >= rows) return;
  typename Pack<T, W>::vec next[V];
  own.load(next, in + row * in_stride);
  float w[V][W], b[V][W];
  own.weights(w, weight, 1.0f);
  own.weights(b, bias, 0.0f);
  for (; row < rows; row += step) {
    float x[V][W];
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int k = 0; k < W; ++k) x[v][k] = (float)next[v][k];
    if (row + step < rows) own.load(next, in + (row + step) * in_stride);
    float m = row_sum<LANES>(own.sum([&](int v, int k) { return x[v][k]; }), lds[0]) / (float)columns;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int k = 0; k < W; ++k) x[v][k] -= m;
    float variance =
        row_sum<LANES>(own.sum([&](int v, int k) { return x[v][k] * x[v][k]; }), lds[1]) / (float)columns;
    if (far_from_zero<LANES>(m, variance)) {  // the same in all threads of a row
      const float rest =
          row_sum<LANES>(own.sum([&](int v, int k) { return x[v][k]; }), lds[2]) / (float)columns;
      m += rest;
      variance = less_rest(variance, rest);
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int k = 0; k < W; ++k) x[v][k] -= rest;
    }
    const float r = 1.0f / sqrtf(variance + epsilon);
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int k = 0; k < W; ++k) x[v][k] = x[v][k] * r * w[v][k] + b[v][k];
    own.store(out + row * out_stride, x);
    if (row_lane<LANES>() == 0) {
      if (mean != nullptr) mean[row] = m;
      if (rstd != nullptr) rstd[row] = r;
    }
  }
}

// Rows too long for the registers: a block reads each of them three times, the second and
// third time from the caches.  The rest of the mean is added up beside the squares (64 x 40000
// bfloat16 11.4 us, 11.2 without; 12.0 by a fourth reading of rows that ask for it).
constexpr int kLongBlock = kWholeBlock;
template <typename T, typename TW>
__global__ __launch_bounds__(kLongBlock) void layer_norm_long_kernel(
    const T* in, int64_t rows, int64_t columns, int64_t in_stride, const TW* __restrict__ weight,
    const TW* __restrict__ bias, float epsilon, T* out, int64_t out_stride,
    float* __restrict__ mean, float* __restrict__ rstd) {
  constexpr int W = 16 / sizeof(T);
  __shared__ float lds[3][kLongBlock / kWaveSize];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* x = in + row * in_stride;
    T* y = out + row * out_stride;
    float sum = 0.0f;
    for (int64_t c = (int64_t)threadIdx.x * W; c < columns; c += kLongBlock * W) {
      float v[W], part = 0.0f;
      load_floats<T, W>(v, x + c, columns - c);
#pragma unroll
      for (int k = 0; k < W; ++k) part += v[k];
      sum += part;
    }
    const float m = row_sum<kLongBlock>(sum, lds[0]) / (float)columns;
    float squares = 0.0f;
    sum = 0.0f;
    for (int64_t c = (int64_t)threadIdx.x * W; c < columns; c += kLongBlock * W) {
      float v[W], part = 0.0f, part_squares = 0.0f;
      load_floats<T, W>(v, x + c, columns - c);
#pragma unroll
      for (int k = 0; k < W; ++k) {
        const float away = c + k < columns ? v[k] - m : 0.0f;
        part += away;
        part_squares += away * away;
      }
      sum += part;
      squares += part_squares;
    }
    put_wave(lanes_sum<kWaveSize>(sum), lds[1]);
    put_wave(lanes_sum<kWaveSize>(squares), lds[2]);
    __syncthreads();
    float rest = sum_waves(lds[1]) / (float)columns;
    float variance = sum_waves(lds[2]) / (float)columns;
    if (far_from_zero<kLongBlock>(m, variance)) variance = less_rest(variance, rest);
    else rest = 0.0f;
    const float r = 1.0f / sqrtf(variance + epsilon), shift = -rest * r;
    for (int64_t c = (int64_t)threadIdx.x * W; c < columns; c += kLongBlock * W) {
      float v[W], w[W], b[W];
      load_floats<T, W>(v, x + c, columns - c);
      if (weight != nullptr) load_floats<TW, W>(w, weight + c, columns - c);
      if (bias != nullptr) load_floats<TW, W>(b, bias + c, columns - c);
#pragma unroll
      for (int k = 0; k < W; ++k) {
        v[k] = fmaf(v[k] - m, r, shift) * (weight != nullptr ? w[k] : 1.0f);
        if (bias != nullptr) v[k] += b[k];
      }
      store_floats<T, W>(y + c, v, columns - c);
    }
    if (threadIdx.x == 0) {
      if (mean != nullptr) mean[row] = m + rest;
      if (rstd != nullptr) rstd[row] = r;
    }
  }
}

// The gradients. A wave or block goes over rows like the forward pass and adds up
// grad_out * h and grad_out of its columns in registers on the way, so the gradient of the
// weights costs no second reading: each block leaves one row of `partials` (blocks x
// columns for the weight, then as many for the bias), which the fold kernel adds up in the
// order of the blocks. A single block writes the results itself.
//
// Fewer waves leave fewer partials, and with the next row on its way they keep the memory
// as busy (waves wanted a compute unit, 32768 x 4096 bfloat16, us: 12 141, 16 151, 32 163; 8192 x
// 1024 15.7, 20.0, 30.8; odd lengths want 12 rather than 8: 3000 columns 83, 95; 16384 x
// 3500 with 14 rather than 7: 74, 105). 32768 x 4096 is 805 MB in 141 us, 5.7 TB/s.
constexpr int kGradientBlock = 512;       // of rows that a wave or a part of one holds
constexpr int kGradientWavesPerCu = 12;
constexpr int kMaxSplitsPerCu = 4;
// Rows a block at least before a compute unit has two (bfloat16, us, 4 / 1: 1000 rows of 1500 12.0
// / 19.5, 600 of 2880 12.9 / 16.4, 1000 of 3500 15.9 / 20.3; with 8, 4000 of 2432 25.1 instead of 21.6).
constexpr int kRowsPerSplit = 4;
template <int LANES> constexpr int gradient_block() {
  return LANES <= kWaveSize ? kGradientBlock : LANES;
}

template <typename T, typename TW, int W, int LANES, int V>
__global__ __launch_bounds__(gradient_block<LANES>()) void layer_norm_gradient_kernel(
    const T* grad_out, int64_t grad_out_stride, const T* in, int64_t in_stride, int64_t rows,
    int64_t columns, const TW* __restrict__ weight, const float* __restrict__ mean,
    const float* __restrict__ rstd, T* grad_in, int64_t grad_in_stride,
    float* __restrict__ partials, int32_t accumulate, TW* __restrict__ grad_weight,
    TW* __restrict__ grad_bias) {
  constexpr int kRows = LANES <= kWaveSize ? kGradientBlock / LANES : 1;  // at a time
  constexpr int kJoins = LANES <= kWaveSize ? kGradientBlock / kWaveSize : 1;
  // The next row on its way costs registers that a large block does not have.
  constexpr bool kAhead = LANES * V * W < 1024 * 16;
  __shared__ float lds[2][2][kMostWaves];
  __shared__ float joined[kJoins > 1 ? kJoins : 1][kJoins > 1 ? LANES * V * W : 1];
  const Columns<W, LANES, V> own(columns);
  const int64_t step = (int64_t)gridDim.x * kRows;
  int64_t row = (int64_t)blockIdx.x * kRows + row_of_block<LANES>();
  float w[V][W], sum_w[V][W], sum_b[V][W];
  own.weights(w, weight, 1.0f);
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int k = 0; k < W; ++k) sum_w[v][k] = sum_b[v][k] = 0.0f;
  typename Pack<T, W>::vec next_x[V], next_g[V];
  float next_m = 0.0f, next_r = 0.0f;
  const auto fetch = [&](int64_t i) {
    own.load(next_x, in + i * in_stride);
    own.load(next_g, grad_out + i * grad_out_stride);
    next_m = mean[i];
    next_r = rstd[i];
  };
  if (kAhead && row < rows) fetch(row);
  for (int turn = 0; row < rows; row += step, turn ^= 1) {
    float h[V][W], g[V][W];
    if (!kAhead) fetch(row);
    const float m = next_m, r = next_r;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int k = 0; k < W; ++k) {
        h[v][k] = ((float)next_x[v][k] - m) * r;
        g[v][k] = (float)next_g[v][k];
        sum_w[v][k] += g[v][k] * h[v][k];
        sum_b[v][k] += g[v][k];
        g[v][k] *= w[v][k];
      }
    if (kAhead && row + step < rows) fetch(row + step);
    if (grad_in == nullptr) continue;
    constexpr int kTogether = LANES <= kWaveSize ? LANES : kWaveSize;
    float mean_g = lanes_sum<kTogether>(own.sum([&](int v, int k) { return g[v][k]; }));
    float mean_gh = lanes_sum<kTogether>(own.sum([&](int v, int k) { return g[v][k] * h[v][k]; }));
    if (LANES > kWaveSize) {
      put_wave(mean_g, lds[turn][0]);
      put_wave(mean_gh, lds[turn][1]);
      __syncthreads();
      mean_g = sum_waves(lds[turn][0]);
      mean_gh = sum_waves(lds[turn][1]);
    }
    mean_g /= (float)columns;
    mean_gh /= (float)columns;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int k = 0; k < W; ++k) h[v][k] = r * (g[v][k] - mean_g - h[v][k] * mean_gh);
    own.store(grad_in + row * grad_in_stride, h);
  }
  if (partials == nullptr) return;
  join_columns<TW, W, LANES, V, kJoins>(own, sum_w, columns, partials + (int64_t)blockIdx.x * columns,
                                        grad_weight, accumulate, joined);
  join_columns<TW, W, LANES, V, kJoins>(own, sum_b, columns,
                                        partials + ((int64_t)gridDim.x + blockIdx.x) * columns,
                                        grad_bias, accumulate, joined);
}

// Rows too long for the registers: a block a row for grad_in, and the columns' sums apart.
template <typename T, typename TW>
__global__ __launch_bounds__(kLongBlock) void layer_norm_long_grad_in_kernel(
    const T* grad_out, int64_t grad_out_stride, const T* in, int64_t in_stride, int64_t rows,
    int64_t columns, const TW* __restrict__ weight, const float* __restrict__ mean,
    const float* __restrict__ rstd, T* grad_in, int64_t grad_in_stride) {
  constexpr int W = 16 / sizeof(T);
  __shared__ float lds[2][kLongBlock / kWaveSize];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* x = in + row * in_stride;
    const T* dy = grad_out + row * grad_out_stride;
    T* dx = grad_in + row * grad_in_stride;
    const float m = mean[row], r = rstd[row];
    const auto load = [&](float (&g)[W], float (&h)[W], int64_t c) {
      load_floats<T, W>(g, dy + c, columns - c);
      load_floats<T, W>(h, x + c, columns - c);
      float w[W];
      if (weight != nullptr) load_floats<TW, W>(w, weight + c, columns - c);
#pragma unroll
      for (int k = 0; k < W; ++k) {
        if (weight != nullptr) g[k] *= w[k];
        h[k] = c + k < columns ? (h[k] - m) * r : 0.0f;
      }
    };
    float sum_g = 0.0f, sum_gh = 0.0f;
    for (int64_t c = (int64_t)threadIdx.x * W; c < columns; c += kLongBlock * W) {
      float g[W], h[W];
      load(g, h, c);
#pragma unroll
      for (int k = 0; k < W; ++k) {
        sum_g += g[k];
        sum_gh += g[k] * h[k];
      }
    }
    const float mean_g = row_sum<kLongBlock>(sum_g, lds[0]) / (float)columns;
    const float mean_gh = row_sum<kLongBlock>(sum_gh, lds[1]) / (float)columns;
    for (int64_t c = (int64_t)threadIdx.x * W; c < columns; c += kLongBlock * W) {
      float g[W], h[W];
      load(g, h, c);
#pragma unroll
      for (int k = 0; k < W; ++k) g[k] = r * (g[k] - mean_g - h[k] * mean_gh);
      store_floats<T, W>(dx + c, g, columns - c);
    }
  }
}

// Block (x, y): columns [256 x, 256 x + 256) over every gridDim.y-th row from y on.
template <typename T>
__global__ __launch_bounds__(kBlock) void layer_norm_column_sums_kernel(
    const T* __restrict__ grad_out, int64_t grad_out_stride, const T* __restrict__ in,
    int64_t in_stride, int64_t rows, int64_t columns, const float* __restrict__ mean,
    const float* __restrict__ rstd, float* __restrict__ partials) {
  const int64_t c = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  if (c >= columns) return;
  float sum_w = 0.0f, sum_b = 0.0f;
#pragma unroll 4
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    const float dy = (float)grad_out[row * grad_out_stride + c];
    sum_w += dy * (((float)in[row * in_stride + c] - mean[row]) * rstd[row]);
    sum_b += dy;
  }
  partials[blockIdx.y * columns + c] = sum_w;
  partials[((int64_t)gridDim.y + blockIdx.y) * columns + c] = sum_b;
}

// Rows of partials at most: one for each block of a launch.
inline int64_t max_splits() { return (int64_t)device_cu_count() * kMaxSplitsPerCu; }
inline int64_t partial_rows(int64_t rows) { return rows < max_splits() ? rows : max_splits(); }

}  // namespace

int32_t launch_layer_norm(hipStream_t stream, const LayerNormArgs& a) {
  if (a.rows == 0) return ILGPU_HIP_SUCCESS;
  return with_norm_types(a.type, a.weight_type, [&](auto t, auto tw) -> int32_t {
    using T = decltype(t);
    using TW = decltype(tw);
    const auto launch = [&](auto kernel, int64_t blocks, int threads) -> int32_t {
      {
        ProfileScope scope(stream, "layer_norm");
        hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(threads), 0, stream,
                           static_cast<const T*>(a.in), a.rows, a.columns, a.in_stride,
                           static_cast<const TW*>(a.weight), static_cast<const TW*>(a.bias),
                           a.epsilon, static_cast<T*>(a.out), a.out_stride, a.mean, a.rstd);
      }
      ILGPU_HIP_CHECK(hipGetLastError());
      return ILGPU_HIP_SUCCESS;
    };
    return with_shape<T>(
        a.columns, kSingleVectors,
        [&](auto w, auto lanes, auto v, int row_threads) {
          constexpr int kLanes = decltype(lanes)::value;
          const int threads = kLanes == kWholeBlock ? row_threads : kBlock;
          const int64_t blocks = div_up(a.rows, block_rows<kLanes>());
          const int64_t most = (int64_t)device_cu_count() * (kWavesPerCu * kWaveSize / threads);
          return launch(
              layer_norm_kernel<T, TW, decltype(w)::value, kLanes, decltype(v)::value>,
              blocks < most ? blocks : most, threads);
        },
        [&] {
          return launch(layer_norm_long_kernel<T, TW>,
                        a.rows < kMaxLongBlocks ? a.rows : kMaxLongBlocks, kLongBlock);
        });
  });
}

int64_t layer_norm_gradient_temp_bytes(int64_t rows, int64_t columns) {
  return 2 * partial_rows(rows) * columns * 4 + 16;
}

int32_t launch_layer_norm_gradient(hipStream_t stream, const LayerNormGradientArgs& a) {
  float* partials = reinterpret_cast<float*>(align_up((int64_t)(uintptr_t)a.temp, 16));
  const bool sums = a.grad_weight != nullptr || a.grad_bias != nullptr;
  return with_norm_types(a.type, a.weight_type, [&](auto t, auto tw) -> int32_t {
    using T = decltype(t);
    using TW = decltype(tw);
    const T* grad_out = static_cast<const T*>(a.grad_out);
    const T* in = static_cast<const T*>(a.in);
    const TW* weight = static_cast<const TW*>(a.weight);
    T* grad_in = static_cast<T*>(a.grad_in);
    const auto fold = [&](int64_t splits) -> int32_t {
      if (!sums) return ILGPU_HIP_SUCCESS;
      const int64_t blocks = div_up(a.columns, kWaveSize);
      for (int64_t first = 0; first < blocks; first += kMaxFoldBlocks) {
        const int64_t some = blocks - first < kMaxFoldBlocks ? blocks - first : kMaxFoldBlocks;
        {
          ProfileScope scope(stream, "layer_norm_fold");
          hipLaunchKernelGGL((fold_partials_kernel<TW>), dim3((unsigned)some, 2),
                             dim3(kFoldBlock), 0, stream, partials, splits, a.columns,
                             a.accumulate, static_cast<TW*>(a.grad_weight),
                             static_cast<TW*>(a.grad_bias), (uint32_t)first);
        }
        ILGPU_HIP_CHECK(hipGetLastError());
      }
      return ILGPU_HIP_SUCCESS;
    };
    if (a.rows == 0) return fold(0);
    return with_shape<T>(
        a.columns, kWholeBlock,
        [&](auto w, auto lanes, auto v, int row_threads) -> int32_t {
          constexpr int kLanes = decltype(lanes)::value;
          const int threads = kLanes == kWholeBlock ? row_threads : kGradientBlock;
          const int64_t blocks =
              div_up(a.rows, kLanes == kWholeBlock ? 1 : kGradientBlock / kLanes);
          // The blocks that come nearest to the waves wanted, of two numbers the smaller.
          int64_t per_cu = (kGradientWavesPerCu * kWaveSize + threads / 2 - 1) / threads;
          // (A block's sums are worth writing after a few rows only.)
          while (per_cu > 1 && a.rows < device_cu_count() * per_cu * kRowsPerSplit) --per_cu;
          per_cu = per_cu < 1 ? 1 : per_cu < kMaxSplitsPerCu ? per_cu : kMaxSplitsPerCu;
          const int64_t most = device_cu_count() * per_cu;
          // (Four turns of one block take less than the fold's launch.)
          const int64_t splits = blocks <= 4 ? 1 : blocks < most ? blocks : most;
          {
            ProfileScope scope(stream, "layer_norm_gradient");
            hipLaunchKernelGGL(
                (layer_norm_gradient_kernel<T, TW, decltype(w)::value, kLanes, decltype(v)::value>),
                dim3((unsigned)splits), dim3(threads), 0, stream, grad_out, a.grad_out_stride, in,
                a.in_stride, a.rows, a.columns, weight, a.mean, a.rstd, grad_in, a.grad_in_stride,
                sums ? partials : nullptr, a.accumulate, static_cast<TW*>(a.grad_weight),
                static_cast<TW*>(a.grad_bias));
          }
          ILGPU_HIP_CHECK(hipGetLastError());
          return splits > 1 ? fold(splits) : ILGPU_HIP_SUCCESS;
        },
        [&]() -> int32_t {
          // The column sums come first: grad_in may be written over what they read.
          if (sums) {
            const int64_t splits = partial_rows(a.rows) < 256 ? partial_rows(a.rows) : 256;
            {
              ProfileScope scope(stream, "layer_norm_column_sums");
              hipLaunchKernelGGL((layer_norm_column_sums_kernel<T>),
                                 dim3((unsigned)div_up(a.columns, kBlock), (unsigned)splits),
                                 dim3(kBlock), 0, stream, grad_out, a.grad_out_stride, in,
                                 a.in_stride, a.rows, a.columns, a.mean, a.rstd, partials);
            }
            ILGPU_HIP_CHECK(hipGetLastError());
            const int32_t rc = fold(splits);
            if (rc != ILGPU_HIP_SUCCESS) return rc;
          }
          if (grad_in != nullptr) {
            ProfileScope scope(stream, "layer_norm_grad_in");
            hipLaunchKernelGGL((layer_norm_long_grad_in_kernel<T, TW>),
                               dim3((unsigned)(a.rows < kMaxLongBlocks ? a.rows : kMaxLongBlocks)),
                               dim3(kLongBlock), 0, stream, grad_out, a.grad_out_stride, in,
                               a.in_stride, a.rows, a.columns, weight, a.mean, a.rstd, grad_in,
                               a.grad_in_stride);
          }
          ILGPU_HIP_CHECK(hipGetLastError());
          return ILGPU_HIP_SUCCESS;
        });
  });
}

}  // namespace ilgpu_hip
