// What the operators on the rows of a matrix share: sums over the threads of a row, a thread's
// columns, the shapes of blocks, and the fold of column sums.
#pragma once

#include "elements.hpp"

namespace ilgpu_hip {
namespace {

constexpr int kBlock = 256;

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
// Blocks of a launch of such: a grid holds less than 2^32 threads along an axis.  They go on to further rows.
constexpr int64_t kMaxLongBlocks = 1 << 20;
static_assert(kMaxLongBlocks * kWholeBlock < INT64_C(1) << 32, "threads of a grid");
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

// The largest block, and the rows it has at a time.
template <int LANES> constexpr int row_block() { return LANES <= kWaveSize ? kBlock : LANES; }
template <int LANES> constexpr int block_rows() { return LANES <= kWaveSize ? kBlock / LANES : 1; }
constexpr int kMostWaves = kWholeBlock / kWaveSize;

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

// The column sums of a block: over the rows of a wave, then over the waves, in their order; into
// the block's row of partials, or, of a single block, to where they belong (result, which may be
// nullptr).  `joined` is LDS of one row of floats for each wave, where more waves than one share the columns.
template <typename TW, int W, int LANES, int V, int WAVES, typename Joined>
__device__ __forceinline__ void join_columns(const Columns<W, LANES, V>& own, float (&sum)[V][W],
                                             int64_t columns, float* to, TW* result,
                                             int32_t accumulate, Joined& joined) {
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
  if constexpr (WAVES > 1) {
    const int wave = threadIdx.x / kWaveSize, lane = threadIdx.x & (kWaveSize - 1);
    if (lane < LANES) {
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int k = 0; k < W; ++k) joined[wave][(v * W + k) * LANES + lane] = sum[v][k];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < LANES * V * W; i += WAVES * kWaveSize) {
      float total = joined[0][i];
#pragma unroll
      for (int j = 1; j < WAVES; ++j) total += joined[j][i];
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
}

// Adds up `splits` rows of partials: 64 columns a block, whose waves take every 16th row;
// blockIdx.y: the weight's, the bias's.  A launch begins at block `first_block`: a grid holds less
// than 2^32 threads, which 2^28 columns would be.
constexpr int kFoldBlock = 1024;
constexpr int64_t kMaxFoldBlocks = 1 << 20;
template <typename TW>
__global__ __launch_bounds__(kFoldBlock) void fold_partials_kernel(
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

}  // namespace
}  // namespace ilgpu_hip
