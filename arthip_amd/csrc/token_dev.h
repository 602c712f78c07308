// Device helpers of the transformer operators: element types and their conversions,
// chunks of values from memory of any element alignment.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/arthip.h"
#include "wino_dev.h"

namespace arthip {

typedef __bf16 b8 __attribute__((ext_vector_type(8)));

// fp32 -> the element type, to nearest even. The arithmetic stays in fp32; this is
// the one rounding of a result.
template <class T>
__device__ __forceinline__ T to_elem(float x) {
  return static_cast<T>(x);
}

// N consecutive values, aligned to an element only: global loads and stores of up to
// 16 bytes take any element alignment on gfx950, at the cost of the extra cache lines
// they touch.
template <class T, int N>
using Vec = T __attribute__((ext_vector_type(N)));

template <class T, int N>
__device__ __forceinline__ void load_chunk(const T* p, float (&out)[N]) {
  if constexpr (N == 1) {
    out[0] = static_cast<float>(*p);
  } else {
    Vec<T, N> c;
    __builtin_memcpy(&c, p, sizeof(c));
    const Vec<float, N> x = __builtin_convertvector(c, Vec<float, N>);
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = x[i];
  }
}

template <class T, int N>
__device__ __forceinline__ void store_chunk(T* p, const float (&x)[N]) {
  if constexpr (N == 1) {
    *p = to_elem<T>(x[0]);
  } else {
    Vec<float, N> v;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = x[i];
    const Vec<T, N> c = __builtin_convertvector(v, Vec<T, N>);
    __builtin_memcpy(p, &c, sizeof(c));
  }
}

}  // namespace arthip
