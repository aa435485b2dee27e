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
#include "elements.hpp"
#include "operators.hpp"

namespace ilgpu_hip {

namespace {

constexpr int kBlock = 256;
constexpr int64_t kMaxBlocks = 1 << 22;

// v moved between lanes by a DPP control, zeros where none comes in; rows of 16 lanes that
// `rows` does not name get zeros too.
template <int CONTROL, int ROWS = 0xf> __device__ __forceinline__ float moved(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CONTROL,
                                                               ROWS, 0xf, true));
}

// The sum over LANES neighbouring lanes (8, 16, 32 or the wave), in all of them, in a fixed
// order.
template <int LANES> __device__ __forceinline__ float lanes_sum(float v) {
  if constexpr (LANES == kWaveSize) {
    v += moved<0x111>(v);       // row_shr:1, 2, 4, 8: a row's sum in its last lane
    v += moved<0x112>(v);
    v += moved<0x114>(v);
    v += moved<0x118>(v);
    v += moved<0x142, 0xa>(v);  // row_bcast:15 into rows 1 and 3
    v += moved<0x143, 0xc>(v);  // row_bcast:31 into rows 2 and 3
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
  } else {
    v += moved<0xb1>(v);                     // quad_perm [1,0,3,2]
    v += moved<0x4e>(v);                     // quad_perm [2,3,0,1]
    v += moved<0x141>(v);                    // row_half_mirror
    if (LANES > 8) v += moved<0x140>(v);     // row_mirror
    if (LANES > 16) v += __shfl_xor(v, 16, kWaveSize);
    return v;
  }
}

// LANES is the number of lanes of a wave that share a row (8, 16, 32, 64), or kWholeBlock: all
// threads of a block do, as many as the row's length asks for.
constexpr int kWholeBlock = 1024;
template <int LANES> __device__ __forceinline__ int row_lanes() {
  return LANES == kWholeBlock ? blockDim.x : LANES;
}
// A thread's place in its row, and its row among those a block has at a time.
template <int LANES> __device__ __forceinline__ int row_lane() {
  return LANES == kWholeBlock ? threadIdx.x : threadIdx.x & (LANES - 1);
}
template <int LANES> __device__ __forceinline__ int row_of_block() {
  if (LANES == kWholeBlock) return 0;
  const int row = threadIdx.x / LANES;
  return LANES == kWaveSize ? __builtin_amdgcn_readfirstlane(row) : row;
}

// The sum over a block's waves of what each has in all of its lanes, in all threads. `slot` is
// LDS of one float per wave (16 at most) that no thread still reads.
__device__ __forceinline__ void put_wave(float v, float* slot) {
  if ((threadIdx.x & (kWaveSize - 1)) == 0) slot[threadIdx.x / kWaveSize] = v;
}
__device__ __forceinline__ float sum_waves(const float* slot) {
  const int i = threadIdx.x & 15;
  return lanes_sum<16>(i < (int)(blockDim.x / kWaveSize) ? slot[i] : 0.0f);
}

// The sum over the threads that share a row, in all of them; a row's sums take slots in turn.
template <int LANES> __device__ __forceinline__ float row_sum(float v, float* slot) {
  if constexpr (LANES <= kWaveSize) {
    return lanes_sum<LANES>(v);
  } else {
    put_wave(lanes_sum<kWaveSize>(v), slot);
    __syncthreads();
    return sum_waves(slot);
  }
}

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

// The columns of a thread: V times W side by side, W times the row's lanes apart.  Where a row ends
// inside a thread's W columns, the thread reads the last W of the row and leaves those of
// its neighbour (`skip` of them; W: all) alone, so every load is whole; columns >= W.
template <int W, int LANES, int V> struct Columns {
  int64_t at[V];
  int skip[V];
  bool whole[V];  // every thread has W of its own
  __device__ __forceinline__ explicit Columns(int64_t columns) {
    const int lane = row_lane<LANES>(), lanes = row_lanes<LANES>();
#pragma unroll
    for (int v = 0; v < V; ++v) {
      whole[v] = (int64_t)(v + 1) * lanes * W <= columns;
      const int64_t c = (int64_t)(v * lanes + lane) * W;
      at[v] = c + W <= columns ? c : columns - W;
      skip[v] = (int)(c - at[v] < W ? c - at[v] : W);
    }
  }
  template <typename T>
  __device__ __forceinline__ void load(typename Pack<T, W>::vec (&r)[V], const T* row) const {
#pragma unroll
    for (int v = 0; v < V; ++v)
      r[v] = *reinterpret_cast<const typename Pack<T, W>::type*>(row + at[v]);
  }
  // (Past the L2, which belongs to one of eight groups of compute units: the next reader is
  // mostly on another. 32768 x 4096 99.9 to 98.1 us, 4099 x 1537 9.3 to 8.7.)
  template <typename T> __device__ __forceinline__ void store(T* row, const float (&y)[V][W]) const {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (skip[v] == 0) {
        typename Pack<T, W>::vec r;
#pragma unroll
        for (int k = 0; k < W; ++k) r[k] = (T)y[v][k];
        __builtin_nontemporal_store(r, reinterpret_cast<typename Pack<T, W>::type*>(row + at[v]));
      } else {
#pragma unroll
        for (int k = 0; k < W; ++k)
          if (k >= skip[v]) row[at[v] + k] = (T)y[v][k];
      }
    }
  }
  // The sum of f(v, k) over the thread's columns.
  template <typename F> __device__ __forceinline__ float sum(F f) const {
    float all = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float part = 0.0f;
      if (whole[v]) {
#pragma unroll
        for (int k = 0; k < W; ++k) part += f(v, k);
      } else {
#pragma unroll
        for (int k = 0; k < W; ++k) part += k >= skip[v] ? f(v, k) : 0.0f;
      }
      all += part;
    }
    return all;
  }
  // A vector of the columns' weights, `otherwise` where there is none.
  template <typename T>
  __device__ __forceinline__ void weights(float (&w)[V][W], const T* p, float otherwise) const {
    if (p != nullptr) {
      typename Pack<T, W>::vec r[V];
      load(r, p);
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int k = 0; k < W; ++k) w[v][k] = (float)r[v][k];
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int k = 0; k < W; ++k) w[v][k] = otherwise;
    }
  }
};

// Blocks of a launch, in waves a compute unit: twice as many as are resident, so that the
// last rows are spread (32768 x 4096, us: 104.6 with 32, 99.9 with 64, 99.7 with 128, 124
// with a block for every row, which loads its weights for it alone; that is what a few thousand
// rows get).
constexpr int kWavesPerCu = 64;

// Rows of more vectors have two in a thread (32768 x 4096: 512 vectors by 256 threads 98 us, by
// 512 101.7).
constexpr int kSingleVectors = 384;

// The largest block, and the rows it has at a time.
template <int LANES> constexpr int row_block() { return LANES <= kWaveSize ? kBlock : LANES; }
template <int LANES> constexpr int block_rows() { return LANES <= kWaveSize ? kBlock / LANES : 1; }
constexpr int kMostWaves = kWholeBlock / kWaveSize;

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

// How a row of `columns` elements of T is shared: by 8 to 64 lanes, or by a block of as many
// waves as its length asks for, each thread with V vectors.  Idle lanes and waves cost like
// others (gradients of bfloat16, us: 2^20 rows of 64 by a wave 461, by 8 lanes 80; 21440 rows of
// 2368 by six waves 78, by five 71).  Calls f(W, LANES, V, threads) with integral constants but for
// `threads`, which is the block's, or `otherwise` for rows beyond; V is 1 up to `single`
// vectors.
template <typename T, typename F, typename G>
int32_t with_shape(int64_t columns, int64_t single, F f, G otherwise) {
  constexpr int W = 16 / sizeof(T);
  const auto shape = [&](auto w, auto lanes, auto v, int64_t vectors) {
    return f(w, lanes, v, (int)align_up(div_up(vectors, decltype(v)::value), kWaveSize));
  };
  using std::integral_constant;
#define ILGPU_HIP_SHAPE(w, lanes, v) \
  shape(integral_constant<int, w>(), integral_constant<int, lanes>(), integral_constant<int, v>(), vectors)
  const int64_t vectors = div_up(columns, W);
  if (columns < W) return ILGPU_HIP_SHAPE(1, 8, 1);
  if (vectors <= 8) return ILGPU_HIP_SHAPE(W, 8, 1);
  if (vectors <= 16) return ILGPU_HIP_SHAPE(W, 16, 1);
  if (vectors <= 32) return ILGPU_HIP_SHAPE(W, 32, 1);
  if (vectors <= 64) return ILGPU_HIP_SHAPE(W, 64, 1);
  if (vectors <= 128) return ILGPU_HIP_SHAPE(W, 64, 2);
  if (vectors <= single) return ILGPU_HIP_SHAPE(W, kWholeBlock, 1);
  if (vectors <= 2048) return ILGPU_HIP_SHAPE(W, kWholeBlock, 2);
  if constexpr (W == 4) {
    if (vectors <= 4096) return ILGPU_HIP_SHAPE(W, kWholeBlock, 4);
  }
#undef ILGPU_HIP_SHAPE
  return otherwise();
}

// Weights have the rows' type or float32.
template <typename F> int32_t with_norm_types(int32_t type, int32_t weight_type, F f) {
  return with_type(type, [&](auto t) -> int32_t {
    if (weight_type == type) return f(t, t);
    return f(t, float());
  });
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
  // The block's sums: over the rows of a wave, then over the waves, in their order; into its
  // row of partials, or, of a single block, to where they belong.
  const auto join = [&](float (&sum)[V][W], float* to, TW* result) {
    const auto put = [&](int64_t c, float total) {
      if (gridDim.x > 1) to[c] = total;
      else if (result != nullptr) result[c] = (TW)(accumulate ? (float)result[c] + total : total);
    };
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int k = 0; k < W; ++k)
#pragma unroll
        for (int off = LANES; off < kWaveSize; off <<= 1)
          sum[v][k] += __shfl_xor(sum[v][k], off, kWaveSize);
    if constexpr (kJoins > 1) {
      const int wave = threadIdx.x / kWaveSize, lane = threadIdx.x & (kWaveSize - 1);
      if (lane < LANES) {
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
          for (int k = 0; k < W; ++k) joined[wave][(v * W + k) * LANES + lane] = sum[v][k];
      }
      __syncthreads();
      for (int i = threadIdx.x; i < LANES * V * W; i += gradient_block<LANES>()) {
        float total = joined[0][i];
#pragma unroll
        for (int j = 1; j < kJoins; ++j) total += joined[j][i];
        const int k = i / LANES % W;
        const int64_t first = ((int64_t)(i / (LANES * W)) * LANES + i % LANES) * W;
        const int64_t at = first + W <= columns ? first : columns - W;
        if (at + k >= first) put(at + k, total);
      }
      __syncthreads();
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int k = 0; k < W; ++k)
          if (k >= own.skip[v]) put(own.at[v] + k, sum[v][k]);
    }
  };
  join(sum_w, partials + (int64_t)blockIdx.x * columns, grad_weight);
  join(sum_b, partials + ((int64_t)gridDim.x + blockIdx.x) * columns, grad_bias);
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

// Adds up `splits` rows of partials: 64 columns a block, whose waves take every 16th row;
// blockIdx.y: the weight's, the bias's.  A launch begins at block `first_block`: a grid holds less
// than 2^32 threads, which 2^28 columns would be.
constexpr int kFoldBlock = 1024;
constexpr int64_t kMaxFoldBlocks = 1 << 20;
template <typename TW>
__global__ __launch_bounds__(kFoldBlock) void layer_norm_fold_kernel(
    const float* __restrict__ partials, int64_t splits, int64_t columns, int32_t accumulate,
    TW* __restrict__ grad_weight, TW* __restrict__ grad_bias, uint32_t first_block) {
  constexpr int kWaves = kFoldBlock / kWaveSize;
  __shared__ float lds[kWaves][kWaveSize];
  TW* to = blockIdx.y == 0 ? grad_weight : grad_bias;
  if (to == nullptr) return;
  const int wave = threadIdx.x / kWaveSize, lane = threadIdx.x & (kWaveSize - 1);
  const int64_t c = (int64_t)(first_block + blockIdx.x) * kWaveSize + lane;
  const float* from = partials + blockIdx.y * splits * columns + c;
  float sum = 0.0f;
  if (c < columns) {
#pragma unroll 8
    for (int64_t s = wave; s < splits; s += kWaves) sum += from[s * columns];
  }
  lds[wave][lane] = sum;
  __syncthreads();
  if (wave != 0 || c >= columns) return;
  for (int i = 1; i < kWaves; ++i) sum += lds[i][lane];
  to[c] = (TW)(accumulate ? (float)to[c] + sum : sum);
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
          return launch(layer_norm_long_kernel<T, TW>, a.rows < kMaxBlocks ? a.rows : kMaxBlocks,
                        kLongBlock);
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
          hipLaunchKernelGGL((layer_norm_fold_kernel<TW>), dim3((unsigned)some, 2),
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
                               dim3((unsigned)(a.rows < kMaxBlocks ? a.rows : kMaxBlocks)),
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
