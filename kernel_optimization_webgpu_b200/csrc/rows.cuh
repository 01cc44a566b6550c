// What the operators over rows of logits share: values and their order.
#pragma once

#include <type_traits>

#include <cuda_bf16.h>

#include "common.cuh"

namespace qd {

// Larger value, larger key; NaN lowest.
__device__ __forceinline__ uint32_t row_key(float v) {
  if (v != v) return 0u;
  const uint32_t u = __float_as_uint(v + 0.0f);  // -0 as +0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float row_key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

template <typename T>
__device__ __forceinline__ float rows_value(const void* p, long long i) {
  if constexpr (sizeof(T) == 4) return static_cast<const float*>(p)[i];
  else if constexpr (std::is_same<T, __half>::value) return __half2float(static_cast<const __half*>(p)[i]);
  else return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

}  // namespace qd
