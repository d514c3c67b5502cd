// The turns of rotary positions: angles, and which values of a head turn together.
#pragma once
#include <hip/hip_runtime.h>

#include "attn_kernels.hpp"

namespace cqgdn {

__device__ __forceinline__ void turn(uint64_t fraction, float& s, float& c) {
  const int32_t hi = (int32_t)(fraction >> 32);
  const uint32_t quadrant = ((uint32_t)hi + 0x20000000u) >> 30;
  // the rest after whole quadrants, in +-1/8 turn
  const float x = (float)(int32_t)((uint32_t)hi - (quadrant << 30)) * 1.46291807926715968e-9f;  // 2 pi / 2^32
  const float z = x * x;
  const float sp =
      x + x * z * (-1.f / 6 + z * (1.f / 120 + z * (-1.f / 5040 + z * (1.f / 362880))));
  const float cp = 1.f + z * (-0.5f + z * (1.f / 24 + z * (-1.f / 720 + z * (1.f / 40320 + z * (-1.f / 3628800)))));
  const float a = (quadrant & 1) ? cp : sp, b = (quadrant & 1) ? sp : cp;
  s = (quadrant & 2) ? -a : a;
  c = ((quadrant + 1) & 2) ? -b : b;
}

// Two vectors of VEC values of one head, one of either half of the values that turn (or of those that pass): lanes
// side by side read side by side in both.
template <int VEC, bool ADJ>
struct TurnPlace {
  int at0, at1;
  bool rot;
  __device__ __forceinline__ TurnPlace(const RotaryArgs& a, int u, int turned) : rot(u < turned) {
    at0 = rot ? u * (ADJ && VEC == 1 ? 2 : VEC) : a.rotary + (u - turned) * VEC;
    at1 = at0 + (rot ? (ADJ && VEC == 1 ? 1 : a.rotary / 2) : (a.D - a.rotary) / 2);
  }
  // the first pair of the vectors' j-th run of RUN pairs
  static constexpr int RUN = ADJ && VEC > 1 ? VEC / 2 : VEC;
  static __device__ __forceinline__ int pair(const RotaryArgs& a, int u, int j) { return u * RUN + (j ? a.rotary / 4 : 0); }
};

__device__ __forceinline__ void angle(const RotaryArgs& a, int64_t t, int pair, float& s, float& c) {
  const int ax = min(max(a.axis[pair], 0), a.axes - 1);
  const int64_t at = ax * a.axis_stride + t;
  const int64_t p = a.wide ? static_cast<const int64_t*>(a.positions)[at]
                           : (int64_t)static_cast<const int32_t*>(a.positions)[at];
  turn((uint64_t)p * a.turns[pair], s, c);
  if (a.back) s = -s;
}

}  // namespace cqgdn
