// exp and the logistic function as the operators' gates take them.
#pragma once

#include "elements.hpp"

namespace ilgpu_hip {

// 2^(x / ln 2) of an x that was a T.  The roundings of the product and of 1 / ln 2 put the result off by
// up to x and x / 5 units of 2^-24: of a float both are put right, of the 16-bit types, whose own last place
// is thousands of times that, they are not.  FINITE: below 2^126, so that its reciprocal is a normal number.
template <typename T, bool FINITE> __device__ __forceinline__ float power_of_e(float x) {
  constexpr float kLog2E = 1.44269504f, kLog2ERest = 1.92596299e-8f;  // 1 / ln 2 to 49 bits
  const float raw = x * kLog2E, t = FINITE && raw > 125.0f ? 125.0f : raw;  // (a NaN stays one)
  const float e = __builtin_amdgcn_exp2f(t);
  if constexpr (!std::is_same<T, float>::value) return e;
  // (Where t was held back, or is infinite, the rest says nothing, and is held to 1.)
  const float rest =
      __builtin_amdgcn_fmed3f(fmaf(x, kLog2ERest, fmaf(x, kLog2E, -t)), -1.0f, 1.0f);
  return e * fmaf(rest, 0.693147181f, 1.0f);
}

// The logistic function of x and what is left of it to 1: 1 / (1 + e) and e / (1 + e) with
// e = exp(-x), each with its own digits.
template <typename T> __device__ __forceinline__ void logistic(float x, float& value, float& left) {
  const float e = power_of_e<T, true>(-x);
  value = __builtin_amdgcn_rcpf(1.0f + e);
  left = e * value;
}

template <typename T> __device__ __forceinline__ float exp_of(float x) {
  return power_of_e<T, false>(x);
}

}  // namespace ilgpu_hip
