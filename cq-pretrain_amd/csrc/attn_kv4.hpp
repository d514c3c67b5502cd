// The 4-bit values of the cache as MFMA operands.
#pragma once
#include "attn_kernels.hpp"
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

// ---- shared by the attention kernels ----------------------------------------------------------------
// The maximum of a row's scores that its weights are taken against need not be the exact one.  It is taken from
// the first positions that the row sees, and moves only where a lane's 16 weights of a step sum to more than
// kAttendLimit.  With fp16 a weight may pass the largest number there (65504).  With bf16 the limit bounds the sums
// of n positions by n 2^12 times the largest value (n times it bounds any softmax's sum before the division), so
// that values up to 2^100 meet no overflow over 2^16 positions, up to 2^84 over any number.
// P is held 2^bias higher because v_exp_f32 drops results below 2^-126 and fp16 keeps 2^-24 at the least:
// weights down to 2^-134 of the maximum count with bf16 (whose results reach 2^-126), down to 2^-31 with fp16.
template <class E>
constexpr float kAttendBias = std::is_same<E, f16>::value ? 7.f : 8.f;
template <class E>
constexpr float kAttendLimit = std::is_same<E, f16>::value ? 60000.f : 65536.f;

// The positions [lo, hi) that a row with the limit `visible` sees of the `room` that its table holds, [0, 0) for
// none.  The window is counted from the limit, which may lie beyond the table.
__device__ __forceinline__ void attend_limits(int visible, int window, int room, int& lo, int& hi) {
  const int limit = max(visible, 0);
  lo = window > 0 ? max(0, limit - window) : 0;
  hi = min(limit, room);
  if (lo >= hi) lo = hi = 0;
}

}  // namespace cqgdn
