// Element types of the operators (float, _Float16, __bf16), wide accesses at
// element alignment and the dispatch from type codes to types.
#pragma once

#include "common.hpp"

namespace ilgpu_hip {

using half_t = _Float16;
using bfloat_t = __bf16;

// -1 for a type the operators do not take (elem_size knows no BF16, so that the
// primitives refuse it).
inline int operator_elem_size(int32_t type) {
  switch (type) {
    case ILGPU_HIP_F32: return 4;
    case ILGPU_HIP_F16: case ILGPU_HIP_BF16: return 2;
    default: return -1;
  }
}

// N elements of T that are aligned like one: gfx950 loads and stores 16 bytes
// from any element's address with one instruction, so rows of odd widths and
// views from the middle of an array take the same path as aligned ones.
template <typename T, int N> struct Pack {
  typedef T vec __attribute__((ext_vector_type(N)));
  typedef vec type __attribute__((aligned(sizeof(T))));
};

// Elements [0, count) of p as floats, zeros from there to N (nothing beyond is read);
// one wide load where all N are there.
template <typename T, int N>
__device__ __forceinline__ void load_floats(float (&v)[N], const T* p, int64_t count) {
  using P = typename Pack<T, N>::type;
  if (count >= N) {
    const P r = *reinterpret_cast<const P*>(p);
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = (float)r[k];
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = k < count ? (float)p[k] : 0.0f;
  }
}

// The first `count` of N floats to p, each rounded to T (nearest even).
template <typename T, int N>
__device__ __forceinline__ void store_floats(T* p, const float (&v)[N], int64_t count) {
  using P = typename Pack<T, N>::type;
  if (count >= N) {
    typename Pack<T, N>::vec r;
#pragma unroll
    for (int k = 0; k < N; ++k) r[k] = (T)v[k];
    *reinterpret_cast<P*>(p) = r;
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (k < count) p[k] = (T)v[k];
  }
}

// x * scale as it is rounded to T next.  (Of a product that is rounded to half the compiler
// makes a fused one with an addend of +0, which turns -0 into +0; the empty statement keeps
// the two apart.)
template <typename T> __device__ __forceinline__ float product_for(float x, float scale) {
  float v = x * scale;
  if constexpr (std::is_same<T, half_t>::value) asm("" : "+v"(v));
  return v;
}

// Calls f(T()) with the element type of a validated type code.
template <typename F> int32_t with_type(int32_t type, F f) {
  switch (type) {
    case ILGPU_HIP_F32: return f(float());
    case ILGPU_HIP_F16: return f(half_t());
    case ILGPU_HIP_BF16: return f(bfloat_t());
    default: return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  }
}
// The same for token numbers.
template <typename F> int32_t with_token_type(int32_t type, F f) {
  switch (type) {
    case ILGPU_HIP_I32: return f(int32_t());
    case ILGPU_HIP_I64: return f(int64_t());
    default: return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  }
}

}  // namespace ilgpu_hip
