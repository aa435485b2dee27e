// One step of AdamW over a list of tensors, with moments in 32 bits or in 8.
//
// The lists go to the kernel by value, as many tensors a launch as fit into 4 KB of arguments, cut
// into chunks of equal length, so tensors of any lengths fill the chip together.  The clip's
// factor and the corrections of the moments come from device memory and are made in every block while its
// loads are on their way.
//
// Moments in 8 bits share a scale, the largest of 256, which a wave holds four in each lane: it decodes
// them, steps, finds the new largest over its lanes and encodes again.  The first stands for the square of its code,
// the second for its fourth power (its root, which the step divides by, for the square), so small
// values keep four and a half digits below the largest.
//
// Bound by the memory in 32 bits: 285 million parameters in float32 with gradients and copies in
// bfloat16 are 8.0 GB in 1412 us, 5.7 TB/s (of 4096 elements a block; 2048 1421 us, 8192 1455).  In 8 bits, where
// they are 16 bytes an element, by the operations of the codes next to it: 90 million 302 us, 4.8 TB/s, with 63
// registers and eight waves a SIMD (seven 320).
#include "elements.hpp"
#include "operators.hpp"

namespace ilgpu_hip {

namespace {

constexpr int kBlock = 256;
constexpr int kW = 4;                         // elements of a thread side by side
static_assert(kW * kWaveSize == kMomentBlock, "a wave has the moments of one scale");
constexpr int kTurn = kBlock * kW;            // elements of a block at a time
// Turns of a chunk, all of whose loads are on their way together.
constexpr int kShortTurns = 2, kLongTurns = 4;
// Elements of a list from which 32 bits take long chunks: 0.5 million in short ones 7.6 us, in long ones
// 8.8 (a quarter of the compute units), 285 million 1421 and 1412.
constexpr int64_t kLongFrom = 1 << 22;
constexpr int kBlocksPerCu = 40;              // of 8 bits: each makes a table of powers
constexpr int kReadTurns = 4;
constexpr int kReadChunk = kReadTurns * kTurn;
constexpr int kTensors = 46;                  // per launch
constexpr int64_t kMaxBlocks = 1 << 22;

struct StepTable {
  void* parameter[kTensors];
  const void* gradient[kTensors];
  void* first[kTensors];
  void* second[kTensors];
  float* first_scale[kTensors];
  float* second_scale[kTensors];
  void* copy[kTensors];
  int64_t length[kTensors];
  uint32_t chunks_end[kTensors];              // chunks of this and all tensors before it
  uint32_t number[kTensors];                  // in the list
  int32_t types[kTensors];                    // of parameter, gradient and copy, 8 bits each
  int32_t count;
};
struct StepNumbers {
  double log_beta1, log_beta2;
  const int64_t* step;
  const float* schedule;
  const float* norm;
  float rate, keep1, keep2, new1, new2, epsilon, weight_decay, max_norm;
  uint32_t seed_low, seed_high;
};
static_assert(sizeof(StepTable) + sizeof(StepNumbers) <= 4000, "kernel arguments");

template <typename Table> __device__ __forceinline__ int tensor_of(const Table& table, uint32_t chunk) {
  int low = 0, high = table.count - 1;
  while (low < high) {
    const int middle = (low + high) >> 1;
    if (table.chunks_end[middle] <= chunk) low = middle + 1;
    else high = middle;
  }
  return low;
}

// Four elements of any of the three types as they lie in memory: the loads of several can be on
// their way, whatever their types, before the first is made a float.
struct Raw {
  uint32_t w[4];
};
typedef uint32_t Words2 __attribute__((ext_vector_type(2)));
typedef uint32_t Words4 __attribute__((ext_vector_type(4)));
typedef Words2 Words2At2 __attribute__((aligned(2)));
typedef Words4 Words4At4 __attribute__((aligned(4)));

__device__ __forceinline__ Raw load_raw(const void* p, int32_t type, int64_t at) {
  Raw r{};
  if (type == ILGPU_HIP_F32) {
    const Words4 v = __builtin_nontemporal_load(
        reinterpret_cast<const Words4At4*>(static_cast<const float*>(p) + at));
    r.w[0] = v[0];
    r.w[1] = v[1];
    r.w[2] = v[2];
    r.w[3] = v[3];
  } else {
    const Words2 v = __builtin_nontemporal_load(
        reinterpret_cast<const Words2At2*>(static_cast<const uint16_t*>(p) + at));
    r.w[0] = v[0];
    r.w[1] = v[1];
  }
  return r;
}
// Elements [0, count) of them.
__device__ __forceinline__ Raw load_some(const void* p, int32_t type, int64_t at, int count) {
  Raw r{};
#pragma unroll
  for (int k = 0; k < kW; ++k) {
    if (k >= count) break;
    if (type == ILGPU_HIP_F32) r.w[k] = static_cast<const uint32_t*>(p)[at + k];
    else r.w[k / 2] |= (uint32_t) static_cast<const uint16_t*>(p)[at + k] << (k % 2 * 16);
  }
  return r;
}
__device__ __forceinline__ void to_floats(float (&v)[kW], const Raw& r, int32_t type) {
  if (type == ILGPU_HIP_F32) {
#pragma unroll
    for (int k = 0; k < kW; ++k) v[k] = __builtin_bit_cast(float, r.w[k]);
  } else if (type == ILGPU_HIP_F16) {
#pragma unroll
    for (int k = 0; k < kW; ++k)
      v[k] = (float)__builtin_bit_cast(half_t, (uint16_t)(r.w[k / 2] >> (k % 2 * 16)));
  } else {
#pragma unroll
    for (int k = 0; k < kW; ++k)
      v[k] = __builtin_bit_cast(float, k % 2 != 0 ? r.w[k / 2] & 0xffff0000u : r.w[k / 2] << 16);
  }
}
template <typename T>
__device__ __forceinline__ void store_as(void* p, int64_t at, const float (&v)[kW], int count) {
  using P = typename Pack<T, kW>::type;
  T* to = static_cast<T*>(p) + at;
  if (count >= kW) {
    typename Pack<T, kW>::vec r;
#pragma unroll
    for (int k = 0; k < kW; ++k) r[k] = (T)v[k];
    __builtin_nontemporal_store(r, reinterpret_cast<P*>(to));
  } else {
#pragma unroll
    for (int k = 0; k < kW; ++k)
      if (k < count) to[k] = (T)v[k];
  }
}
__device__ __forceinline__ void store_any(void* p, int32_t type, int64_t at, const float (&v)[kW],
                                          int count) {
  if (type == ILGPU_HIP_F32) store_as<float>(p, at, v, count);
  else if (type == ILGPU_HIP_F16) store_as<half_t>(p, at, v, count);
  else store_as<bfloat_t>(p, at, v, count);
}

// What is the same for all elements of a step.
struct Step {
  float factor, back;                      // of the gradients, one after the other
  float rate, keep;                        // r / (1 - beta1^t), 1 - r * weight_decay
  float inverse2;                          // 1 / (1 - beta2^t)
  bool finite;
};
__device__ __forceinline__ Step step_of(const StepNumbers& n) {
  Step s;
  s.factor = s.back = 1.0f;
  s.finite = true;
  if (n.norm != nullptr) {
    const float norm = n.norm[0];
    s.finite = fabsf(norm) <= 3.402823466e+38f;
    if (norm > n.max_norm) {
      // A factor below the normal numbers has few bits: it is made 2^120 times as large and taken
      // back behind the product.
      const bool tiny = n.max_norm / norm < 0x1p-126f;
      s.factor = tiny ? n.max_norm * 0x1p120f / norm : n.max_norm / norm;
      s.back = tiny ? 0x1p-120f : 1.0f;
    }
  }
  const float rate = n.schedule != nullptr ? n.rate * n.schedule[0] : n.rate;
  const double t = (double)n.step[0];
  s.rate = rate / -expm1f((float)(t * n.log_beta1));
  s.inverse2 = 1.0f / -expm1f((float)(t * n.log_beta2));
  s.keep = fmaf(-rate, n.weight_decay, 1.0f);
  return s;
}

// One element's step from its moments, which become the new ones; returns the new parameter.
__device__ __forceinline__ float stepped(const StepNumbers& n, const Step& s, float p, float gradient,
                                         float& m, float& v) {
  {
    // (Each rounded by itself: see first_value.)
#pragma clang fp contract(off)
    const float g = gradient * s.factor * s.back;
    m = n.keep1 * m + n.new1 * g;
    v = n.keep2 * v + n.new2 * (g * g);
  }
  const float root = __builtin_amdgcn_sqrtf(v * s.inverse2) + n.epsilon;
  return fmaf(s.keep, p, -s.rate * m * __builtin_amdgcn_rcpf(root));
}

// A hash of a 32-bit number: xor-shifts and products with odd numbers (the first bits of the fractions of
// the roots of 2 and 3), each of which can be undone, so no two numbers share a hash.
__host__ __device__ __forceinline__ uint32_t mixed(uint32_t x) {
  x ^= x >> 16;
  x *= 0x6a09e667u;
  x ^= x >> 15;
  x *= 0xbb67ae85u;
  return x ^ (x >> 16);
}

// The largest of a wave's lanes, of numbers whose order is that of their bits (none negative; a
// NaN is larger than all).
template <int CONTROL, int ROWS = 0xf> __device__ __forceinline__ uint32_t moved_bits(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CONTROL, ROWS, 0xf, true);
}
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ float wave_largest(float x) {
  uint32_t v = __builtin_bit_cast(uint32_t, x);
  v = larger(v, moved_bits<0x111>(v));       // row_shr:1, 2, 4, 8
  v = larger(v, moved_bits<0x112>(v));
  v = larger(v, moved_bits<0x114>(v));
  v = larger(v, moved_bits<0x118>(v));
  v = larger(v, moved_bits<0x142, 0xa>(v));  // row_bcast:15 into rows 1 and 3
  v = larger(v, moved_bits<0x143, 0xc>(v));  // row_bcast:31 into rows 2 and 3
  return __builtin_bit_cast(float, (uint32_t)__builtin_amdgcn_readlane((int)v, 63));
}
__device__ __forceinline__ float larger_bits(float a, float b) {
  return __builtin_bit_cast(float, larger(__builtin_bit_cast(uint32_t, a),
                                          __builtin_bit_cast(uint32_t, b)));
}

// What codes stand for.  Which of two codes a value near a border gets is decided by its last bit, and
// the next steps go on from there, so the order of roundings is a part of the format: the code's
// power, the scale's part and their product, each rounded to float32 by itself, the power by the
// library's function, as a program that computes in whole arrays does it.
constexpr float kFirstUnit = 1.0f / (127.0f * 127.0f);
constexpr float kSecondUnit = 1.0f / (255.0f * 255.0f * 255.0f * 255.0f);
__device__ __forceinline__ float first_value(uint32_t code, float unit) {  // unit: scale * kFirstUnit
  const float q = (float)(int)code - 128.0f;
  return q * fabsf(q) * unit;
}
// The fourth powers of all codes, in LDS.
using Powers = float[256];
__device__ __forceinline__ void fill_powers(Powers& powers) {
  static_assert(kBlock == 256, "a thread a code");
  powers[threadIdx.x] = powf((float)threadIdx.x, 4.0f);
  __syncthreads();
}

// The code of a value that is not negative: the last whose value is not above it, or the next one
// if `chance` / 2^16 of the way to it is less than the rest.  The share of the scale is a quotient rounded to
// float32, everything behind it exact (float64, in which the products with powers are as good as that).
template <int POWER> struct Code {
  static constexpr float kLevels = POWER == 2 ? 127.0f : 255.0f;
  static constexpr double kAll = POWER == 2 ? 127.0 * 127.0 : 255.0 * 255.0 * 255.0 * 255.0;
  static __device__ __forceinline__ double power(float code) {
    const double square = (double)(code * code);  // (exact in float32)
    return POWER == 2 ? square : square * square;
  }
  static __device__ __forceinline__ float root(float z) {
    z = __builtin_amdgcn_sqrtf(z);
    return POWER == 2 ? z : __builtin_amdgcn_sqrtf(z);
  }
  static __device__ float exactly(float value, float scale, uint32_t chance) {
    const double z = (double)(value / scale) * kAll;
    float low = floorf(root((float)z));
    double below = power(low), way = z - below, span = power(low + 1.0f) - below;
    if (way < 0.0 || way >= span) {  // (the root's roundings)
      low += way < 0.0 ? -1.0f : 1.0f;
      below = power(low);
      way = z - below;
      span = power(low + 1.0f) - below;
    }
    return fminf(low + (way > (double)chance * 0x1p-16 * span ? 1.0f : 0.0f), kLevels);
  }
  // The same in float32; `sure` becomes false where its roundings might decide: z is off by 5 units of 2^-24 of
  // it at most (the reciprocal by 2, the two products and the quotient of the exact way by one each), the rest by
  // less than another.  Or where the root's might (another 12 units of z): `low` is then next to a code's value
  // and one too large or too small, and the code is the same, one that is raised or the next that is not, unless
  // chance / 2^16 of the way between two codes, z / 64 at least, is less than those 17 units: below 5, or that far
  // from 2^16.  (90 million moments with both in float64 378 us, bound by its operations.)
  static __device__ __forceinline__ float nearly(float value, float inverse, uint32_t chance, bool& sure) {
    const float z = value * inverse, low = floorf(root(z));  // inverse: (float)kAll / scale
    const float step = fmaf(2.0f, low, 1.0f), square = low * low;
    float way, span;
    if constexpr (POWER == 2) {
      way = fmaf(-low, low, z);
      span = step;
    } else {
      way = fmaf(-square, square, z);
      span = step * fmaf(2.0f, square, step);
    }
    const float rest = fmaf(-0x1p-16f * (float)chance, span, way);
    sure = sure && fabsf(rest) > z * 4e-7f && chance - 5u < 65527u;
    return low + (rest > 0.0f ? 1.0f : 0.0f);
  }
};
// Scales below the first are none: all codes are those of zero.  The reciprocals of those above the second
// are below the normal numbers, and the instruction may give 0 for them: their codes are made exactly.
constexpr float kSmallest = 0x1p-126f, kLargest = 0x1p126f;

typedef uint32_t WordAt1 __attribute__((aligned(1)));
__device__ __forceinline__ uint32_t load_codes(const void* p, int64_t at, int count) {
  const uint8_t* from = static_cast<const uint8_t*>(p) + at;
  if (count >= kW) return *reinterpret_cast<const WordAt1*>(from);
  uint32_t w = 0;
#pragma unroll
  for (int k = 0; k < kW; ++k)
    if (k < count) w |= (uint32_t)from[k] << (8 * k);
  return w;
}
__device__ __forceinline__ void store_codes(void* p, int64_t at, uint32_t w, int count) {
  uint8_t* to = static_cast<uint8_t*>(p) + at;
  if (count >= kW) {
    *reinterpret_cast<WordAt1*>(to) = w;
    return;
  }
#pragma unroll
  for (int k = 0; k < kW; ++k)
    if (k < count) to[k] = (uint8_t)(w >> (8 * k));
}

template <bool EIGHT, int TURNS>
__global__ __launch_bounds__(kBlock, EIGHT ? 8 : 4) void adamw_kernel(StepTable table, StepNumbers numbers) {
  __shared__ Powers powers;
  if (EIGHT) fill_powers(powers);
  constexpr int kTurns = TURNS, kChunk = TURNS * kTurn;
  const uint32_t chunks = table.chunks_end[table.count - 1];
  Step s;
  bool known = false;
  for (uint32_t chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    const int t = tensor_of(table, chunk);
    const int64_t first = (int64_t)(chunk - (t > 0 ? table.chunks_end[t - 1] : 0)) * kChunk;
    const int64_t length = table.length[t];
    const int32_t types = table.types[t];
    const int32_t type_p = types & 255, type_g = types >> 8 & 255, type_c = types >> 16;
    Raw p[kTurns], g[kTurns], m[kTurns], v[kTurns];
    float unit1[kTurns], unit2[kTurns];
#pragma unroll
    for (int u = 0; u < kTurns; ++u) {
      const int64_t at = first + u * kTurn + threadIdx.x * kW, left = length - at;
      if (left >= kW) {
        p[u] = load_raw(table.parameter[t], type_p, at);
        g[u] = load_raw(table.gradient[t], type_g, at);
        if (!EIGHT) {
          m[u] = load_raw(table.first[t], ILGPU_HIP_F32, at);
          v[u] = load_raw(table.second[t], ILGPU_HIP_F32, at);
        }
      } else {
        p[u] = load_some(table.parameter[t], type_p, at, (int)left);
        g[u] = load_some(table.gradient[t], type_g, at, (int)left);
        if (!EIGHT) {
          m[u] = load_some(table.first[t], ILGPU_HIP_F32, at, (int)left);
          v[u] = load_some(table.second[t], ILGPU_HIP_F32, at, (int)left);
        }
      }
      if (EIGHT) {
        const int count = left < kW ? (int)left : kW;
        m[u].w[0] = load_codes(table.first[t], at, count);
        v[u].w[0] = load_codes(table.second[t], at, count);
        const int64_t block = (first + u * kTurn) / kMomentBlock + threadIdx.x / kWaveSize;
        const bool there = block * kMomentBlock < length;
        unit1[u] = there ? table.first_scale[t][block] * kFirstUnit : 0.0f;
        unit2[u] = there ? table.second_scale[t][block] * kSecondUnit : 0.0f;
      }
    }
    if (!known) s = step_of(numbers);  // while the first chunk is on its way
    known = true;
    if (!s.finite) return;
    uint32_t key = 0;
    if (EIGHT) {
      key = mixed(numbers.seed_low + (uint32_t)numbers.step[0] * 0x3c6ef373u);
      key = mixed(key + numbers.seed_high + table.number[t] * 0x9e3779b9u);
    }
#pragma unroll
    for (int u = 0; u < kTurns; ++u) {
      const int64_t at = first + u * kTurn + threadIdx.x * kW;
      const int count = length - at < kW ? (int)(length - at) : kW;
      if (!EIGHT && count <= 0) break;
      float parameter[kW], gradient[kW], moment1[kW], moment2[kW];
      to_floats(parameter, p[u], type_p);
      to_floats(gradient, g[u], type_g);
#pragma unroll
      for (int k = 0; k < kW; ++k) {
        if (EIGHT) {
          moment1[k] = first_value(m[u].w[0] >> (8 * k) & 255u, unit1[u]);
          moment2[k] = powers[v[u].w[0] >> (8 * k) & 255u] * unit2[u];
        } else {
          moment1[k] = __builtin_bit_cast(float, m[u].w[k]);
          moment2[k] = __builtin_bit_cast(float, v[u].w[k]);
        }
        parameter[k] = stepped(numbers, s, parameter[k], gradient[k], moment1[k], moment2[k]);
      }
      if (count > 0) {
        store_any(table.parameter[t], type_p, at, parameter, count);
        if (table.copy[t] != nullptr) store_any(table.copy[t], type_c, at, parameter, count);
      }
      if (!EIGHT) {
        store_as<float>(table.first[t], at, moment1, count);
        store_as<float>(table.second[t], at, moment2, count);
        continue;
      }
      float largest1 = 0.0f, largest2 = 0.0f;
#pragma unroll
      for (int k = 0; k < kW; ++k) {
        if (k < count) {
          largest1 = larger_bits(largest1, fabsf(moment1[k]));
          largest2 = larger_bits(largest2, fabsf(moment2[k]));
        }
      }
      const float scale1 = wave_largest(largest1), scale2 = wave_largest(largest2);
      const float inverse1 = scale1 < kSmallest ? 0.0f : (float)Code<2>::kAll * __builtin_amdgcn_rcpf(scale1);
      const float inverse2 = scale2 < kSmallest ? 0.0f : (float)Code<4>::kAll * __builtin_amdgcn_rcpf(scale2);
      uint32_t codes1 = 0, codes2 = 0;
#pragma unroll
      for (int k = 0; k < kW; ++k) {
        const uint32_t chance = mixed((uint32_t)(at + k) * 0x9e3779b9u + key);
        bool sure = scale1 <= kLargest && scale2 <= kLargest;
        float code1 = Code<2>::nearly(fabsf(moment1[k]), inverse1, chance & 0xffffu, sure);
        float code2 = Code<4>::nearly(moment2[k], inverse2, chance >> 16, sure);
        if (__any(!sure)) {  // (of a hundred waves three)
          code1 = scale1 < kSmallest ? 0.0f : Code<2>::exactly(fabsf(moment1[k]), scale1, chance & 0xffffu);
          code2 = scale2 < kSmallest ? 0.0f : Code<4>::exactly(moment2[k], scale2, chance >> 16);
        }
        codes1 = __builtin_amdgcn_cvt_pk_u8_f32(128.0f + copysignf(code1, moment1[k]), k, codes1);
        codes2 = __builtin_amdgcn_cvt_pk_u8_f32(code2, k, codes2);
      }
      if (count > 0) {
        store_codes(table.first[t], at, codes1, count);
        store_codes(table.second[t], at, codes2, count);
      }
      const int64_t block = (first + u * kTurn) / kMomentBlock + threadIdx.x / kWaveSize;
      if ((threadIdx.x & (kWaveSize - 1)) == 0 && block * kMomentBlock < length) {
        table.first_scale[t][block] = scale1 < kSmallest ? 0.0f : scale1;
        table.second_scale[t][block] = scale2 < kSmallest ? 0.0f : scale2;
      }
    }
  }
}

constexpr int kReadTensors = 90;
struct ReadTable {
  const void* codes[kReadTensors];
  const float* scales[kReadTensors];
  void* target[kReadTensors];
  int64_t length[kReadTensors];
  uint32_t chunks_end[kReadTensors];
  int32_t type[kReadTensors];
  int32_t count;
};
static_assert(sizeof(ReadTable) <= 4000, "kernel arguments");

template <bool SECOND>
__global__ __launch_bounds__(kBlock) void adamw_moments_kernel(ReadTable table) {
  __shared__ Powers powers;
  if (SECOND) fill_powers(powers);
  const uint32_t chunks = table.chunks_end[table.count - 1];
  for (uint32_t chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    const int t = tensor_of(table, chunk);
    const int64_t first = (int64_t)(chunk - (t > 0 ? table.chunks_end[t - 1] : 0)) * kReadChunk;
    uint32_t codes[kReadTurns];
    float unit[kReadTurns];
#pragma unroll
    for (int u = 0; u < kReadTurns; ++u) {
      const int64_t at = first + u * kTurn + threadIdx.x * kW, left = table.length[t] - at;
      codes[u] = load_codes(table.codes[t], at, left < kW ? (int)left : kW);
      unit[u] = left > 0 ? table.scales[t][at / kMomentBlock] * (SECOND ? kSecondUnit : kFirstUnit)
                         : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < kReadTurns; ++u) {
      const int64_t at = first + u * kTurn + threadIdx.x * kW, left = table.length[t] - at;
      if (left <= 0) break;
      float v[kW];
#pragma unroll
      for (int k = 0; k < kW; ++k) {
        const uint32_t code = codes[u] >> (8 * k) & 255u;
        v[k] = SECOND ? powers[code] * unit[u] : first_value(code, unit[u]);
      }
      store_any(table.target[t], table.type[t], at, v, left < kW ? (int)left : kW);
    }
  }
}

}  // namespace

int32_t launch_adamw(hipStream_t stream, const AdamwArgs& a) {
  const ilgpu_hip_adamw_options& o = a.options;
  StepNumbers numbers;
  numbers.log_beta1 = log(o.beta1);
  numbers.log_beta2 = log(o.beta2);
  numbers.step = a.step;
  numbers.schedule = a.schedule;
  numbers.norm = a.norm;
  numbers.rate = (float)o.rate;
  numbers.keep1 = (float)o.beta1;
  numbers.keep2 = (float)o.beta2;
  numbers.new1 = (float)(1.0 - o.beta1);
  numbers.new2 = (float)(1.0 - o.beta2);
  numbers.epsilon = (float)o.epsilon;
  numbers.weight_decay = (float)o.weight_decay;
  numbers.max_norm = (float)o.max_norm;
  numbers.seed_low = (uint32_t)(uint64_t)o.seed;
  numbers.seed_high = (uint32_t)((uint64_t)o.seed >> 32);
  const bool eight = a.first_scales != nullptr;
  int64_t elements = 0;
  for (int64_t k = 0; k < a.count; ++k) elements += a.parameters[k].length;
  const bool long_chunks = !eight && elements >= kLongFrom;
  StepTable table;
  for (int64_t next = 0; next < a.count;) {
    int used = 0;
    int64_t chunks = 0;
    for (; next < a.count && used < kTensors; ++next) {
      const int64_t length = a.parameters[next].length;
      if (length == 0) continue;
      chunks += div_up(length, (long_chunks ? kLongTurns : kShortTurns) * kTurn);  // (at most 2^29 and one per tensor)
      table.parameter[used] = a.parameters[next].data;
      table.gradient[used] = a.gradients[next].data;
      table.first[used] = a.first[next].data;
      table.second[used] = a.second[next].data;
      table.first_scale[used] = eight ? static_cast<float*>(a.first_scales[next].data) : nullptr;
      table.second_scale[used] = eight ? static_cast<float*>(a.second_scales[next].data) : nullptr;
      table.copy[used] = a.copies != nullptr ? a.copies[next].data : nullptr;
      table.length[used] = length;
      table.chunks_end[used] = (uint32_t)chunks;
      table.number[used] = (uint32_t)next;
      table.types[used] = a.parameters[next].type | a.gradients[next].type << 8 |
                          (a.copies != nullptr ? a.copies[next].type << 16 : 0);
      ++used;
    }
    if (used == 0) break;
    table.count = used;
    {
      ProfileScope scope(stream, eight ? "adamw_8bit" : "adamw");
      // (With 8 bits a block that goes on to further chunks has its table of powers for all.)
      const int64_t most = eight ? (int64_t)device_cu_count() * kBlocksPerCu : kMaxBlocks;
      const dim3 grid((unsigned)(chunks < most ? chunks : most));
      const auto kernel = eight ? adamw_kernel<true, kShortTurns>
                                : long_chunks ? adamw_kernel<false, kLongTurns>
                                              : adamw_kernel<false, kShortTurns>;
      hipLaunchKernelGGL(kernel, grid, dim3(kBlock), 0, stream, table, numbers);
    }
    ILGPU_HIP_CHECK(hipGetLastError());
  }
  return ILGPU_HIP_SUCCESS;
}

int32_t launch_adamw_moments(hipStream_t stream, const ilgpu_hip_tensor* codes,
                             const ilgpu_hip_tensor* scales, const ilgpu_hip_tensor* targets,
                             int64_t count, bool second) {
  ReadTable table;
  for (int64_t next = 0; next < count;) {
    int used = 0;
    int64_t chunks = 0;
    for (; next < count && used < kReadTensors; ++next) {
      if (codes[next].length == 0) continue;
      chunks += div_up(codes[next].length, kReadChunk);
      table.codes[used] = codes[next].data;
      table.scales[used] = static_cast<const float*>(scales[next].data);
      table.target[used] = targets[next].data;
      table.length[used] = codes[next].length;
      table.chunks_end[used] = (uint32_t)chunks;
      table.type[used] = targets[next].type;
      ++used;
    }
    if (used == 0) break;
    table.count = used;
    {
      ProfileScope scope(stream, "adamw_moments");
      const dim3 grid((unsigned)(chunks < kMaxBlocks ? chunks : kMaxBlocks));
      if (second)
        hipLaunchKernelGGL((adamw_moments_kernel<true>), grid, dim3(kBlock), 0, stream, table);
      else
        hipLaunchKernelGGL((adamw_moments_kernel<false>), grid, dim3(kBlock), 0, stream, table);
    }
    ILGPU_HIP_CHECK(hipGetLastError());
  }
  return ILGPU_HIP_SUCCESS;
}

}  // namespace ilgpu_hip
