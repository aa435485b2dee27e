// exp and the logistic function as the operators' gates take them.
#pragma once

#include "elements.hpp"

namespace ilgpu_hip {

// exp(x) to about a unit in the last place: of x / ln 2 the part that the product rounds off is
// put right behind the hardware's 2^x.
__device__ __forceinline__ float exp_of(float x) {
  constexpr float kLog2E = 1.44269504f, kLog2ELow = 1.92596299e-8f;  // log2(e) in two parts
  x = x < -150.0f ? -150.0f : x;  // (a NaN stays one)
  x = x > 150.0f ? 150.0f : x;
  const float t = x * kLog2E;
  const float rest = fmaf(x, kLog2ELow, fmaf(x, kLog2E, -t));
  return __builtin_amdgcn_exp2f(t) * fmaf(rest, 0.693147181f, 1.0f);
}

// The logistic function of x and what is left of it to 1, each to some units in its last place: of
// exp(-|x|), which does not overflow, the larger and the smaller of the two.
__device__ __forceinline__ void logistic(float x, float& value, float& left) {
  const float e = exp_of(-fabsf(x));
  const float larger = __builtin_amdgcn_rcpf(1.0f + e), smaller = e * larger;
  value = x >= 0.0f ? larger : smaller;
  left = x >= 0.0f ? smaller : larger;
}

}  // namespace ilgpu_hip
