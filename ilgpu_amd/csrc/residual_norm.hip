// What stands between two blocks: the norm behind the one with its gate, the residual stream and
// the norm in front of the next, and the gradients of it all.
//
// Norms are by the root of the mean square, sums in float32 in a fixed order.  `out` is made from
// the total before it is rounded.
//
// Bound by the memory: a row of every matrix is read once, stays in the registers of the wave
// or block that has it, and every result is written once.  32768 x 2048 bfloat16 with the stream in
// float32: 940 MB in 173 us, 5.4 TB/s; gradients of 16384 x 4096 bfloat16: 1074 MB in 207 us, 5.2 TB/s.
#include "gates.hpp"
#include "operators.hpp"
#include "rows.hpp"

namespace ilgpu_hip {

namespace {

constexpr int kLongBlock = kWholeBlock;

// act(gate), and its slope.  Beyond kFar what is left is below the normal numbers: an infinite gate
// is shut, or open, although infinity times 0 is no number.
constexpr float kFar = 87.0f;
template <typename T> __device__ __forceinline__ float activation(float gate, int32_t kind) {
  float s, left;
  logistic<T>(gate, s, left);
  return kind == ILGPU_HIP_GATE_SIGMOID ? s : gate < -kFar ? 0.0f : gate * s;
}
template <typename T>
__device__ __forceinline__ float activation(float gate, int32_t kind, float& slope) {
  float s, left;
  logistic<T>(gate, s, left);
  const float both = s * left;
  if (kind == ILGPU_HIP_GATE_SIGMOID) {
    slope = both;
    return s;
  }
  slope = fabsf(gate) > kFar ? s : fmaf(gate, both, s);
  return gate < -kFar ? 0.0f : gate * s;
}

template <int W, int LANES, int V, typename T>
__device__ __forceinline__ void any_weights(const Columns<W, LANES, V>& own, float (&w)[V][W],
                                            const void* p, bool wide, T) {
  if (wide) own.weights(w, static_cast<const float*>(p), 1.0f);
  else own.weights(w, static_cast<const T*>(p), 1.0f);
}

template <typename T> __device__ __forceinline__ const T* row_of(const void* p, int64_t row,
                                                                int64_t stride) {
  return static_cast<const T*>(p) + row * stride;
}
template <typename T> __device__ __forceinline__ T* row_of(void* p, int64_t row, int64_t stride) {
  return static_cast<T*>(p) + row * stride;
}

// Two sums of a row, a float for each wave, alternating between rows: what one row's sums are put into is
// read by others until the sums of the row behind it.
using Slots = float[2][2][kMostWaves];

template <typename T, typename TR, int W, int LANES, int V>
__global__ __launch_bounds__(row_block<LANES>()) void residual_norm_kernel(ResidualNormArgs a) {
  constexpr int kRows = block_rows<LANES>();
  __shared__ Slots lds;
  const Columns<W, LANES, V> own(a.columns);
  const int64_t step = (int64_t)gridDim.x * kRows;
  int64_t row = (int64_t)blockIdx.x * kRows + row_of_block<LANES>();
  if (row >= a.rows) return;
  const bool wide = a.weight_type == ILGPU_HIP_F32;
  typename Pack<T, W>::vec next_x[V], next_gate[V];
  typename Pack<TR, W>::vec next_residual[V];
  const auto fetch = [&](int64_t i) {
    own.load(next_x, row_of<T>(a.in, i, a.in_stride));
    if (a.gate != nullptr) own.load(next_gate, row_of<T>(a.gate, i, a.gate_stride));
    if (a.residual != nullptr) own.load(next_residual, row_of<TR>(a.residual, i, a.residual_stride));
  };
  fetch(row);
  float w[V][W], input_w[V][W];
  any_weights(own, w, a.weight, wide, T());
  any_weights(own, input_w, a.input_weight, wide, T());
  const float columns = (float)a.columns;
  for (int turn = 0; row < a.rows; row += step, turn ^= 1) {
    float x[V][W], y[V][W];
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int k = 0; k < W; ++k) {
        x[v][k] = (float)next_x[v][k];
        y[v][k] = a.gate != nullptr ? activation<T>((float)next_gate[v][k], a.gate_kind) : 1.0f;
      }
    float r[V][W];
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int k = 0; k < W; ++k) r[v][k] = a.residual != nullptr ? (float)next_residual[v][k] : 0.0f;
    if (row + step < a.rows) fetch(row + step);
    if (a.input_norm) {
      const float squares =
          row_sum<LANES>(own.sum([&](int v, int k) { return x[v][k] * x[v][k]; }), lds[turn][0]);
      const float rstd = 1.0f / sqrtf(squares / columns + a.epsilon);
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int k = 0; k < W; ++k) x[v][k] = x[v][k] * rstd * input_w[v][k];
      if (a.input_rstd != nullptr && row_lane<LANES>() == 0) a.input_rstd[row] = rstd;
    }
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int k = 0; k < W; ++k) x[v][k] = fmaf(a.scale, x[v][k] * y[v][k], r[v][k]);
    if (a.total != nullptr) own.store(row_of<TR>(a.total, row, a.total_stride), x);
    if (a.out == nullptr && a.rstd == nullptr) continue;
    const float squares =
        row_sum<LANES>(own.sum([&](int v, int k) { return x[v][k] * x[v][k]; }), lds[turn][1]);
    const float rstd = 1.0f / sqrtf(squares / columns + a.epsilon);
    if (a.rstd != nullptr && row_lane<LANES>() == 0) a.rstd[row] = rstd;
    if (a.out == nullptr) continue;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int k = 0; k < W; ++k) x[v][k] = x[v][k] * rstd * w[v][k];
    own.store(row_of<T>(a.out, row, a.out_stride), x);
  }
}

// W weights from column c on, 1 where there are none.
template <typename T, int W>
__device__ __forceinline__ void long_weights(float (&w)[W], const void* p, bool wide, int64_t c,
                                             int64_t count) {
  if (p == nullptr) {
#pragma unroll
    for (int k = 0; k < W; ++k) w[k] = 1.0f;
  } else if (wide) {
    load_floats<float, W>(w, static_cast<const float*>(p) + c, count);
  } else {
    load_floats<T, W>(w, static_cast<const T*>(p) + c, count);
  }
}

// Calls f(column, columns from there to the row's end) for the vectors of a thread of a block that
// has the row.
template <int W, typename F> __device__ __forceinline__ void for_columns(int64_t columns, F f) {
  for (int64_t c = (int64_t)threadIdx.x * W; c < columns; c += (int64_t)blockDim.x * W)
    f(c, columns - c);
}

// Rows too long for the registers: a block a row, which reads it up to three times, from the
// caches but for the first.  Nothing is written before the last reading.
template <typename T, typename TR>
__global__ __launch_bounds__(kLongBlock) void residual_norm_long_kernel(ResidualNormArgs a) {
  constexpr int W = 16 / sizeof(T);
  __shared__ Slots lds;
  const bool wide = a.weight_type == ILGPU_HIP_F32;
  const float columns = (float)a.columns;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    float input_rstd = 1.0f;
    if (a.input_norm) {
      float squares = 0.0f;
      for_columns<W>(a.columns, [&](int64_t c, int64_t count) {
        float x[W], part = 0.0f;
        load_floats<T, W>(x, row_of<T>(a.in, row, a.in_stride) + c, count);
#pragma unroll
        for (int k = 0; k < W; ++k) part += x[k] * x[k];
        squares += part;
      });
      squares = row_sum<kLongBlock>(squares, lds[turn][0]);
      input_rstd = 1.0f / sqrtf(squares / columns + a.epsilon);
      if (a.input_rstd != nullptr && threadIdx.x == 0) a.input_rstd[row] = input_rstd;
    }
    const auto total_at = [&](int64_t c, int64_t count, float (&x)[W]) {
      load_floats<T, W>(x, row_of<T>(a.in, row, a.in_stride) + c, count);
      if (a.input_norm) {
        float w[W];
        long_weights<T, W>(w, a.input_weight, wide, c, count);
#pragma unroll
        for (int k = 0; k < W; ++k) x[k] = x[k] * input_rstd * w[k];
      }
      if (a.gate != nullptr) {
        float gate[W];
        load_floats<T, W>(gate, row_of<T>(a.gate, row, a.gate_stride) + c, count);
#pragma unroll
        for (int k = 0; k < W; ++k) x[k] *= activation<T>(gate[k], a.gate_kind);
      }
      float r[W];
#pragma unroll
      for (int k = 0; k < W; ++k) r[k] = 0.0f;
      if (a.residual != nullptr)
        load_floats<TR, W>(r, row_of<TR>(a.residual, row, a.residual_stride) + c, count);
#pragma unroll
      for (int k = 0; k < W; ++k) x[k] = fmaf(a.scale, x[k], r[k]);
    };
    float rstd = 1.0f;
    if (a.out != nullptr || a.rstd != nullptr) {
      float squares = 0.0f;
      for_columns<W>(a.columns, [&](int64_t c, int64_t count) {
        float x[W], part = 0.0f;
        total_at(c, count, x);
#pragma unroll
        for (int k = 0; k < W; ++k) part += k < count ? x[k] * x[k] : 0.0f;
        squares += part;
      });
      squares = row_sum<kLongBlock>(squares, lds[turn][1]);
      rstd = 1.0f / sqrtf(squares / columns + a.epsilon);
      if (a.rstd != nullptr && threadIdx.x == 0) a.rstd[row] = rstd;
    }
    for_columns<W>(a.columns, [&](int64_t c, int64_t count) {
      float x[W];
      total_at(c, count, x);
      if (a.total != nullptr)
        store_floats<TR, W>(row_of<TR>(a.total, row, a.total_stride) + c, x, count);
      if (a.out == nullptr) return;
      float w[W];
      long_weights<T, W>(w, a.weight, wide, c, count);
#pragma unroll
      for (int k = 0; k < W; ++k) x[k] = x[k] * rstd * w[k];
      store_floats<T, W>(row_of<T>(a.out, row, a.out_stride) + c, x, count);
    });
  }
}

// ---- the gradients ---------------------------------------------------------------------
// A wave or block goes over rows like the forward pass and adds up what its columns give to the
// weights' gradients on the way; a second kernel adds up the blocks' sums in their order.
constexpr int kGradientBlock = 512;
constexpr int kGradientWavesPerCu = 16;
constexpr int kMaxSplitsPerCu = 4;
constexpr int kRowsPerSplit = 4;
// Up to 512 vectors a row, two blocks share a compute unit with 128 registers a thread, so that one loads
// while the other waits for its sums; longer rows have a block for themselves.
constexpr int kWideBlock = 512;

// Waves of a SIMD: as many as leave the registers that a thread asks for.  (16384 x 4096 bfloat16, a block
// of 512 threads a row: 209 us with 128 registers and two blocks a compute unit, 247 with 136 and one;
// with the stream in float32, which 128 registers spill, 152 against 204 with 8192 rows.)
template <typename T, typename TR, int LANES, int V> constexpr int gradient_waves() {
  if (sizeof(T) == 4) return LANES <= kWaveSize && V > 1 ? 3 : 4;
  return V > 1 ? 2 : LANES <= kWaveSize || sizeof(TR) == 4 ? 3 : 4;
}
template <typename T, typename TR, int W, int LANES, int V, int BLOCK>
__global__ __launch_bounds__(BLOCK, (gradient_waves<T, TR, LANES, V>())) void residual_norm_gradient_kernel(
    ResidualNormGradientArgs a, float* __restrict__ partials) {
  constexpr int kRows = LANES <= kWaveSize ? BLOCK / LANES : 1;  // at a time
  constexpr int kJoins = LANES <= kWaveSize ? BLOCK / kWaveSize : 1;
  constexpr bool kAhead = V == 1;
  __shared__ Slots lds;
  __shared__ float joined[kJoins > 1 ? kJoins : 1][kJoins > 1 ? LANES * V * W : 1];
  const Columns<W, LANES, V> own(a.columns);
  const int64_t step = (int64_t)gridDim.x * kRows;
  int64_t row = (int64_t)blockIdx.x * kRows + row_of_block<LANES>();
  const bool wide = a.weight_type == ILGPU_HIP_F32;
  float w[V][W], input_w[V][W], sum_w[V][W], sum_input[V][W];
  any_weights(own, w, a.weight, wide, T());
  any_weights(own, input_w, a.input_weight, wide, T());
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int k = 0; k < W; ++k) sum_w[v][k] = sum_input[v][k] = 0.0f;
  typename Pack<T, W>::vec next_grad[V], next_x[V], next_gate[V];
  typename Pack<TR, W>::vec next_total[V], next_grad_total[V];
  float next_rstd = 0.0f, next_input_rstd = 1.0f;
  const auto fetch = [&](int64_t i) {
    if (a.grad_out != nullptr) {
      own.load(next_grad, row_of<T>(a.grad_out, i, a.grad_out_stride));
      own.load(next_total, row_of<TR>(a.total, i, a.total_stride));
      next_rstd = a.rstd[i];
    }
    if (a.grad_total != nullptr)
      own.load(next_grad_total, row_of<TR>(a.grad_total, i, a.grad_total_stride));
    own.load(next_x, row_of<T>(a.in, i, a.in_stride));
    if (a.gate != nullptr) own.load(next_gate, row_of<T>(a.gate, i, a.gate_stride));
    if (a.input_norm) next_input_rstd = a.input_rstd[i];
  };
  if (kAhead && row < a.rows) fetch(row);
  for (int turn = 0; row < a.rows; row += step, turn ^= 1) {
    if (!kAhead) fetch(row);
    float h[V][W], g[V][W], d[V][W], x[V][W], gate[V][W];
    const float rstd = next_rstd, input_rstd = next_input_rstd;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int k = 0; k < W; ++k) {
        d[v][k] = a.grad_total != nullptr ? (float)next_grad_total[v][k] : 0.0f;
        x[v][k] = (float)next_x[v][k];
        gate[v][k] = a.gate != nullptr ? (float)next_gate[v][k] : 0.0f;
        if (a.grad_out != nullptr) {
          h[v][k] = (float)next_total[v][k] * rstd;
          g[v][k] = (float)next_grad[v][k];
          sum_w[v][k] += g[v][k] * h[v][k];
          g[v][k] *= w[v][k];
        }
      }
    if (kAhead && row + step < a.rows) fetch(row + step);
    if (a.grad_out != nullptr) {
      const float mean = row_sum<LANES>(own.sum([&](int v, int k) { return g[v][k] * h[v][k]; }),
                                        lds[turn][0]) / (float)a.columns;
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int k = 0; k < W; ++k) d[v][k] = fmaf(rstd, g[v][k] - h[v][k] * mean, d[v][k]);
    }
    if (a.grad_residual != nullptr)
      own.store(row_of<TR>(a.grad_residual, row, a.grad_residual_stride), d);
    // From here on d is the gradient of what was added to the stream, x the normalised input.
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int k = 0; k < W; ++k) {
        d[v][k] *= a.scale;
        x[v][k] *= input_rstd;
      }
    if (a.gate != nullptr) {
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int k = 0; k < W; ++k) {
          float slope;
          const float open = activation<T>(gate[v][k], a.gate_kind, slope);
          gate[v][k] = d[v][k] * (x[v][k] * input_w[v][k]) * slope;
          d[v][k] *= open;
        }
      if (a.grad_gate != nullptr)
        own.store(row_of<T>(a.grad_gate, row, a.grad_gate_stride), gate);
    }
    if (a.input_norm) {
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int k = 0; k < W; ++k) {
          sum_input[v][k] += d[v][k] * x[v][k];
          d[v][k] *= input_w[v][k];
        }
      if (a.grad_in != nullptr) {
        const float mean = row_sum<LANES>(own.sum([&](int v, int k) { return d[v][k] * x[v][k]; }),
                                          lds[turn][1]) / (float)a.columns;
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
          for (int k = 0; k < W; ++k) d[v][k] = input_rstd * (d[v][k] - x[v][k] * mean);
      }
    }
    if (a.grad_in != nullptr) own.store(row_of<T>(a.grad_in, row, a.grad_in_stride), d);
  }
  if (partials == nullptr) return;
  float* to = partials + (int64_t)blockIdx.x * a.columns;
  float* to_input = to + (int64_t)gridDim.x * a.columns;
  const auto join = [&](auto type) {
    using TW = decltype(type);
    if (a.grad_weight != nullptr)
      join_columns<TW, W, LANES, V, kJoins>(own, sum_w, a.columns, to, static_cast<TW*>(a.grad_weight),
                                            a.accumulate, joined);
    if (a.grad_input_weight != nullptr)
      join_columns<TW, W, LANES, V, kJoins>(own, sum_input, a.columns, to_input,
                                            static_cast<TW*>(a.grad_input_weight), a.accumulate,
                                            joined);
  };
  if (wide) join(float());
  else join(T());
}

// Rows too long for the registers.  What an element's gradients are made of:
template <typename T, typename TR, int W> struct LongRow {
  const ResidualNormGradientArgs& a;
  int64_t row;
  float rstd, input_rstd;
  bool wide;
  __device__ __forceinline__ LongRow(const ResidualNormGradientArgs& args, int64_t r)
      : a(args), row(r), rstd(args.grad_out != nullptr ? args.rstd[r] : 0.0f),
        input_rstd(args.input_norm ? args.input_rstd[r] : 1.0f),
        wide(args.weight_type == ILGPU_HIP_F32) {}
  // g = grad_out * weight (or grad_out itself) and h = total * rstd.
  __device__ __forceinline__ void of_out(int64_t c, int64_t count, float (&g)[W], float (&h)[W],
                                         bool weighted) const {
#pragma unroll
    for (int k = 0; k < W; ++k) g[k] = h[k] = 0.0f;
    if (a.grad_out == nullptr) return;
    load_floats<T, W>(g, row_of<T>(a.grad_out, row, a.grad_out_stride) + c, count);
    load_floats<TR, W>(h, row_of<TR>(a.total, row, a.total_stride) + c, count);
    float w[W];
    long_weights<T, W>(w, weighted ? a.weight : nullptr, wide, c, count);
#pragma unroll
    for (int k = 0; k < W; ++k) {
      g[k] *= w[k];
      h[k] = k < count ? h[k] * rstd : 0.0f;
    }
  }
  // The gradient of total, from the mean of g * h.
  __device__ __forceinline__ void of_total(int64_t c, int64_t count, float mean, float (&d)[W]) const {
    float g[W], h[W];
    of_out(c, count, g, h, true);
#pragma unroll
    for (int k = 0; k < W; ++k) d[k] = 0.0f;
    if (a.grad_total != nullptr)
      load_floats<TR, W>(d, row_of<TR>(a.grad_total, row, a.grad_total_stride) + c, count);
#pragma unroll
    for (int k = 0; k < W; ++k) d[k] = fmaf(rstd, g[k] - h[k] * mean, d[k]);
  }
  // From d: the gate's gradient, e = d * act(gate) * scale, and x = in * input_rstd.
  __device__ __forceinline__ void of_in(int64_t c, int64_t count, float (&d)[W], float (&x)[W],
                                        float (&of_gate)[W], const float (&input_w)[W]) const {
    load_floats<T, W>(x, row_of<T>(a.in, row, a.in_stride) + c, count);
#pragma unroll
    for (int k = 0; k < W; ++k) {
      d[k] *= a.scale;
      x[k] = k < count ? x[k] * input_rstd : 0.0f;
    }
    if (a.gate == nullptr) return;
    float gate[W];
    load_floats<T, W>(gate, row_of<T>(a.gate, row, a.gate_stride) + c, count);
#pragma unroll
    for (int k = 0; k < W; ++k) {
      float slope;
      const float open = activation<T>(gate[k], a.gate_kind, slope);
      of_gate[k] = d[k] * (x[k] * input_w[k]) * slope;
      d[k] *= open;
    }
  }
};

// The two means of a row.
template <typename T, typename TR>
__global__ __launch_bounds__(kLongBlock) void residual_norm_long_means_kernel(
    ResidualNormGradientArgs a, float* __restrict__ means) {
  constexpr int W = 16 / sizeof(T);
  __shared__ Slots lds;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    const LongRow<T, TR, W> of(a, row);
    float mean = 0.0f, input_mean = 0.0f;
    if (a.grad_out != nullptr) {
      for_columns<W>(a.columns, [&](int64_t c, int64_t count) {
        float g[W], h[W], part = 0.0f;
        of.of_out(c, count, g, h, true);
#pragma unroll
        for (int k = 0; k < W; ++k) part += g[k] * h[k];
        mean += part;
      });
      mean = row_sum<kLongBlock>(mean, lds[turn][0]) / (float)a.columns;
    }
    if (a.input_norm) {
      for_columns<W>(a.columns, [&](int64_t c, int64_t count) {
        float d[W], x[W], of_gate[W], w[W], part = 0.0f;
        long_weights<T, W>(w, a.input_weight, of.wide, c, count);
        of.of_total(c, count, mean, d);
        of.of_in(c, count, d, x, of_gate, w);
#pragma unroll
        for (int k = 0; k < W; ++k) part += k < count ? d[k] * w[k] * x[k] : 0.0f;
        input_mean += part;
      });
      input_mean = row_sum<kLongBlock>(input_mean, lds[turn][1]) / (float)a.columns;
    }
    if (threadIdx.x == 0) {
      means[2 * row] = mean;
      means[2 * row + 1] = input_mean;
    }
  }
}

// Block (x, y): a vector of columns a thread over every gridDim.y-th row from y on.
template <typename T, typename TR>
__global__ __launch_bounds__(kBlock) void residual_norm_long_sums_kernel(
    ResidualNormGradientArgs a, const float* __restrict__ means, float* __restrict__ partials) {
  constexpr int W = 16 / sizeof(T);
  const int64_t c = ((int64_t)blockIdx.x * kBlock + threadIdx.x) * W, count = a.columns - c;
  if (count <= 0) return;
  float sum_w[W], sum_input[W], w[W];
#pragma unroll
  for (int k = 0; k < W; ++k) sum_w[k] = sum_input[k] = 0.0f;
  long_weights<T, W>(w, a.input_weight, a.weight_type == ILGPU_HIP_F32, c, count);
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const LongRow<T, TR, W> of(a, row);
    if (a.grad_weight != nullptr) {
      float g[W], h[W];
      of.of_out(c, count, g, h, false);
#pragma unroll
      for (int k = 0; k < W; ++k) sum_w[k] += g[k] * h[k];
    }
    if (a.grad_input_weight != nullptr) {
      float d[W], x[W], of_gate[W];
      of.of_total(c, count, means[2 * row], d);
      of.of_in(c, count, d, x, of_gate, w);
#pragma unroll
      for (int k = 0; k < W; ++k) sum_input[k] += d[k] * x[k];
    }
  }
  float* to = partials + (int64_t)blockIdx.y * a.columns + c;
  store_floats<float, W>(to, sum_w, count);
  store_floats<float, W>(to + (int64_t)gridDim.y * a.columns, sum_input, count);
}

template <typename T, typename TR>
__global__ __launch_bounds__(kLongBlock) void residual_norm_long_gradient_kernel(
    ResidualNormGradientArgs a, const float* __restrict__ means) {
  constexpr int W = 16 / sizeof(T);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const LongRow<T, TR, W> of(a, row);
    const float mean = means[2 * row], input_mean = means[2 * row + 1];
    for_columns<W>(a.columns, [&](int64_t c, int64_t count) {
      float d[W], x[W], of_gate[W], w[W];
      long_weights<T, W>(w, a.input_weight, of.wide, c, count);
      of.of_total(c, count, mean, d);
      float of_residual[W];
#pragma unroll
      for (int k = 0; k < W; ++k) of_residual[k] = d[k];
      of.of_in(c, count, d, x, of_gate, w);
      if (a.input_norm) {
#pragma unroll
        for (int k = 0; k < W; ++k) d[k] = of.input_rstd * (d[k] * w[k] - x[k] * input_mean);
      }
      if (a.grad_residual != nullptr)
        store_floats<TR, W>(row_of<TR>(a.grad_residual, row, a.grad_residual_stride) + c,
                            of_residual, count);
      if (a.grad_gate != nullptr)
        store_floats<T, W>(row_of<T>(a.grad_gate, row, a.grad_gate_stride) + c, of_gate, count);
      if (a.grad_in != nullptr)
        store_floats<T, W>(row_of<T>(a.grad_in, row, a.grad_in_stride) + c, d, count);
    });
  }
}

inline int64_t max_splits() { return (int64_t)device_cu_count() * kMaxSplitsPerCu; }
inline int64_t partial_rows(int64_t rows) { return rows < max_splits() ? rows : max_splits(); }
constexpr int64_t kLongFrom = 4096;  // columns from which a type's rows may be long ones
constexpr int64_t kLongSplits = 256;

// The matrices' type and the residual stream's.
template <typename F> int32_t with_residual_types(int32_t type, int32_t residual_type, F f) {
  return with_norm_types(type, residual_type, f);
}

}  // namespace

int32_t launch_residual_norm(hipStream_t stream, const ResidualNormArgs& a) {
  if (a.rows == 0) return ILGPU_HIP_SUCCESS;
  // (Waves wanted a compute unit, 32768 x 2048 bfloat16, the stream in float32, us: 32 188, 64 184, 128 177,
  // 512 173: four rows in a block one after the other, whose weights come from the caches each time.)
  constexpr int kWavesPerCu = 512;
  return with_residual_types(a.type, a.residual_type, [&](auto t, auto tr) -> int32_t {
    using T = decltype(t);
    using TR = decltype(tr);
    const auto launch = [&](auto kernel, int64_t blocks, int threads) -> int32_t {
      {
        ProfileScope scope(stream, "residual_norm");
        hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(threads), 0, stream, a);
      }
      ILGPU_HIP_CHECK(hipGetLastError());
      return ILGPU_HIP_SUCCESS;
    };
    return with_shape<T>(
        a.columns, kWholeBlock,
        [&](auto w, auto lanes, auto v, int row_threads) {
          constexpr int kLanes = decltype(lanes)::value;
          const int threads = kLanes == kWholeBlock ? row_threads : kBlock;
          const int64_t blocks = div_up(a.rows, block_rows<kLanes>());
          const int64_t most = (int64_t)device_cu_count() * (kWavesPerCu * kWaveSize / threads);
          return launch(
              residual_norm_kernel<T, TR, decltype(w)::value, kLanes, decltype(v)::value>,
              blocks < most ? blocks : most, threads);
        },
        [&] {
          return launch(residual_norm_long_kernel<T, TR>,
                        a.rows < kMaxLongBlocks ? a.rows : kMaxLongBlocks, kLongBlock);
        });
  });
}

// Partial sums of both weights, and two means for each row of long ones.
int64_t residual_norm_gradient_temp_bytes(int64_t rows, int64_t columns) {
  return 2 * partial_rows(rows) * columns * 4 + (columns > kLongFrom ? 8 * rows : 0) + 16;
}

int32_t launch_residual_norm_gradient(hipStream_t stream, const ResidualNormGradientArgs& a,
                                      void* temp) {
  float* partials = reinterpret_cast<float*>(align_up((int64_t)(uintptr_t)temp, 16));
  const bool sums = a.grad_weight != nullptr || a.grad_input_weight != nullptr;
  return with_residual_types(a.type, a.residual_type, [&](auto t, auto tr) -> int32_t {
    using T = decltype(t);
    using TR = decltype(tr);
    const auto fold = [&](int64_t splits) -> int32_t {
      if (!sums) return ILGPU_HIP_SUCCESS;
      const int64_t blocks = div_up(a.columns, kWaveSize);
      for (int64_t first = 0; first < blocks; first += kMaxFoldBlocks) {
        const int64_t some = blocks - first < kMaxFoldBlocks ? blocks - first : kMaxFoldBlocks;
        const auto launch = [&](auto type) {
          using TW = decltype(type);
          ProfileScope scope(stream, "residual_norm_fold");
          hipLaunchKernelGGL((fold_partials_kernel<TW>), dim3((unsigned)some, 2), dim3(kFoldBlock),
                             0, stream, partials, splits, a.columns, a.accumulate,
                             static_cast<TW*>(a.grad_weight),
                             static_cast<TW*>(a.grad_input_weight), (uint32_t)first);
        };
        if (a.weight_type == ILGPU_HIP_F32) launch(float());
        else launch(T());
        ILGPU_HIP_CHECK(hipGetLastError());
      }
      return ILGPU_HIP_SUCCESS;
    };
    if (a.rows == 0) return fold(0);
    const auto in_registers = [&](auto w, auto lanes, auto v, auto block, int threads) -> int32_t {
      constexpr int kLanes = decltype(lanes)::value;
      const int64_t blocks = div_up(a.rows, kLanes == kWholeBlock ? 1 : kGradientBlock / kLanes);
      int64_t per_cu = (kGradientWavesPerCu * kWaveSize + threads / 2 - 1) / threads;
      while (per_cu > 1 && a.rows < device_cu_count() * per_cu * kRowsPerSplit) --per_cu;
      per_cu = per_cu < 1 ? 1 : per_cu < kMaxSplitsPerCu ? per_cu : kMaxSplitsPerCu;
      const int64_t most = device_cu_count() * per_cu;
      const int64_t splits = blocks <= 4 ? 1 : blocks < most ? blocks : most;
      {
        ProfileScope scope(stream, "residual_norm_gradient");
        hipLaunchKernelGGL((residual_norm_gradient_kernel<T, TR, decltype(w)::value, kLanes,
                                                          decltype(v)::value, decltype(block)::value>),
                           dim3((unsigned)splits), dim3(threads), 0, stream, a,
                           sums ? partials : nullptr);
      }
      ILGPU_HIP_CHECK(hipGetLastError());
      return splits > 1 ? fold(splits) : ILGPU_HIP_SUCCESS;
    };
    const auto of_long_rows = [&]() -> int32_t {
      const int64_t across = div_up(div_up(a.columns, 16 / (int64_t)sizeof(T)), kBlock);
      int64_t splits = partial_rows(a.rows) < kLongSplits ? partial_rows(a.rows) : kLongSplits;
      // (A grid holds less than 2^32 threads.)
      while (splits > 1 && across * splits * kBlock >= INT64_C(1) << 32) splits /= 2;
      const int64_t blocks = a.rows < kMaxLongBlocks ? a.rows : kMaxLongBlocks;
      float* means = partials + 2 * partial_rows(a.rows) * a.columns;
      {
        ProfileScope scope(stream, "residual_norm_means");
        hipLaunchKernelGGL((residual_norm_long_means_kernel<T, TR>), dim3((unsigned)blocks),
                           dim3(kLongBlock), 0, stream, a, means);
      }
      ILGPU_HIP_CHECK(hipGetLastError());
      // The column sums come first: what they read may be written over.
      if (sums) {
        {
          ProfileScope scope(stream, "residual_norm_column_sums");
          hipLaunchKernelGGL((residual_norm_long_sums_kernel<T, TR>),
                             dim3((unsigned)across, (unsigned)splits), dim3(kBlock), 0, stream, a,
                             means, partials);
        }
        ILGPU_HIP_CHECK(hipGetLastError());
        const int32_t rc = fold(splits);
        if (rc != ILGPU_HIP_SUCCESS) return rc;
      }
      {
        ProfileScope scope(stream, "residual_norm_gradient");
        hipLaunchKernelGGL((residual_norm_long_gradient_kernel<T, TR>), dim3((unsigned)blocks),
                           dim3(kLongBlock), 0, stream, a, means);
      }
      ILGPU_HIP_CHECK(hipGetLastError());
      return ILGPU_HIP_SUCCESS;
    };
    using std::integral_constant;
    // A vector a thread in up to 1024 threads where a thread's registers hold the next row beside it; with a
    // wider stream two vectors in up to 512.  (8192 rows bfloat16 by one vector and by two, us: 5120 columns
    // 163 and 189, 8192 213 and 241; with the stream in float32, whose second row spills, 6144 321 and 278.)
    constexpr bool kOneVector = sizeof(T) == sizeof(TR);
    return with_shape<T>(
        a.columns, kOneVector ? kWholeBlock : kWideBlock,
        [&](auto w, auto lanes, auto v, int row_threads) -> int32_t {
          constexpr int kLanes = decltype(lanes)::value, kV = decltype(v)::value;
          const auto block = [&](auto size) { return in_registers(w, lanes, v, size, row_threads); };
          if constexpr (kLanes <= kWaveSize) {
            return in_registers(w, lanes, v, integral_constant<int, kGradientBlock>(), kGradientBlock);
          } else if constexpr (kV > 2 || (kV == 2 && kOneVector && sizeof(T) == 2)) {
            return of_long_rows();
          } else {
            if constexpr (kV == 1 || sizeof(T) == 2)
              if (row_threads <= kWideBlock) return block(integral_constant<int, kWideBlock>());
            if constexpr (kOneVector) return block(integral_constant<int, kWholeBlock>());
            else return of_long_rows();
          }
        },
        of_long_rows);
  });
}

}  // namespace ilgpu_hip
