// What the kernels of the attention's gradients share.
#pragma once
#include "attn_core.hpp"

namespace cqgdn {

constexpr int kGradRows = 128;  // of a workgroup for dq, 32 a wave
// keys of a workgroup for dk and dv
template <int D>
constexpr int kKeys = D == 256 ? 64 : 256;

template <class E>
constexpr float kWeightBias = std::is_same<E, f16>::value ? 15.f : 0.f;

// Two elements of the type from two floats
template <class E>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef E x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x, y}, x2));
}

// dx goes into its product in two bf16 terms, 2^-17 of it, where a mask cuts a step: there lie the rows that see few keys,
// whose dx and gradients are many times those of the others (in 9216 causal rows 2^-9 of the first rows' dx is up to 0.45
// times the root mean square of dq).  In fp16 one term is 2^-12.  (9216 rows: 2% of the gradients' time.)
template <class E, bool WHOLE>
constexpr bool kTwoTerms = !WHOLE && !std::is_same<E, f16>::value;
// what pack2(x, y) = w leaves of x and y
template <class E>
__device__ __forceinline__ uint32_t rest2(float x, float y, uint32_t w) {
  const float a = x - __builtin_bit_cast(float, w << 16), b = y - __builtin_bit_cast(float, w & 0xFFFF0000u);
  return pack2<E>(a - a == 0.f ? a : 0.f, b - b == 0.f ? b : 0.f);
}

// The power of two that a lane's dx go with in fp16 (bf16: 1): the largest lies near 2^10 when it is set, and below
// 2^15 always.  The two lanes of a column share it.
template <class E>
struct Range {
  static constexpr bool on = std::is_same<E, f16>::value;
  float f = on ? 0.f : 1.f;
  // for 16 new dx; `acc`, the sums so far, move with it
  template <int MT>
  __device__ __forceinline__ void fit(const f32x16& x, f32x16 (&acc)[MT]) {
    if constexpr (on) {
      float top = fabsf(x[0]);
#pragma unroll
      for (int e = 1; e < 16; ++e) top = fmaxf(top, fabsf(x[e]));
      bool move = top * f > 32768.f || (f == 0.f && top > 0.f);
      if (__any(move)) {
        move = __shfl_xor((int)move, 32, 64) || move;
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        if (move) {
          const int e = (int)(__builtin_bit_cast(uint32_t, top) >> 23) - 127;
          const float g = __builtin_bit_cast(float, (uint32_t)(127 + min(max(10 - e, -126), 126)) << 23);
          const float by = f == 0.f ? 0.f : g / f;
#pragma unroll
          for (int m = 0; m < MT; ++m) acc[m] *= by;
          f = g;
        }
      }
    }
  }
  // what the sums are to be multiplied with
  __device__ __forceinline__ float back() const { return !on ? 1.f : f == 0.f ? 0.f : 1.f / f; }
};

// dk and dv, in `splits` parts, of the `blocks` blocks of 64 rows that the kernel for dq has left (attn_core_dkv.hip)
template <class E, int D>
void launch_dkv(const CoreGradArgs& a, int blocks, int splits, hipStream_t st);

}  // namespace cqgdn
