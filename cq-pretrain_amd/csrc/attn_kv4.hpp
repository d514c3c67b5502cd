// The 4-bit values of the cache as MFMA operands.
#pragma once
#include "gdn_common.hpp"

namespace cqgdn {

// the scale as the conversion instructions take it (they read the exponent field): byte 255, the
// exponent of infinities and NaN, converts every code to NaN
__device__ __forceinline__ float kv4_scale(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }

// the eight values of a word of codes, in order
template <class E>
__device__ __forceinline__ typename Vec<E>::x8 kv4_values(uint32_t code, float scale);
template <>
__device__ __forceinline__ bf16x8 kv4_values<bf16>(uint32_t code, float scale) {
  const auto a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, scale, 0);
  const auto b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, scale, 1);
  const auto c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, scale, 2);
  const auto d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, scale, 3);
  return __builtin_shufflevector(__builtin_shufflevector(a, b, 0, 1, 2, 3), __builtin_shufflevector(c, d, 0, 1, 2, 3),
                                 0, 1, 2, 3, 4, 5, 6, 7);
}
template <>
__device__ __forceinline__ f16x8 kv4_values<f16>(uint32_t code, float scale) {
  const auto a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(code, scale, 0);
  const auto b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(code, scale, 1);
  const auto c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(code, scale, 2);
  const auto d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(code, scale, 3);
  return __builtin_shufflevector(__builtin_shufflevector(a, b, 0, 1, 2, 3), __builtin_shufflevector(c, d, 0, 1, 2, 3),
                                 0, 1, 2, 3, 4, 5, 6, 7);
}

}  // namespace cqgdn
