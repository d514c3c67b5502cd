// Rotary positions with several axes.
//
// A head's first `rotary` values are pairs; pair i turns by the angle position[axis[i]] * f_i, its
// gradient by the opposite angle.  The frequency comes as turns a position in 64-bit fixed point, so
// the low 64 bits of position * turns are the fraction of a turn, exact for every integer position
// (an fp32 product is off by 0.06 rad at position 10^6).  Its top 32 bits are rounded to the nearest
// eighth of a turn's quadrant and the Taylor polynomials of sine and cosine, degrees 9 and 10 on
// +-pi/4 (remainders 2e-9 and 1e-10), give the rest.
#include <hip/hip_runtime.h>

#include "attn_kernels.hpp"
#include "cqgdn.h"

namespace cqgdn {
namespace {

constexpr int kThreads = 256;
constexpr int kTogether = 4;  // heads whose loads are under way at once

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

// A thread keeps the angles of VEC pairs of one token in registers and takes them through `per` heads, so that
// a sine and cosine (some 40 operations) are paid once for several heads; the loads of kTogether heads go out
// before the first is turned.
template <class T, int VEC, bool ADJ>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a, int units, int turned, int per) {
  const int64_t t = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (t >= a.T) return;
  typedef T P __attribute__((ext_vector_type(VEC)));
  const int all = a.heads[0] + a.heads[1], h0 = blockIdx.y * per, h1 = min(h0 + per, all);
  const T* const xq = static_cast<const T*>(a.x[0]) + t * a.token[0];
  const T* const xk = static_cast<const T*>(a.x[1]) + t * a.token[1];
  T* const yq = static_cast<T*>(a.y[0]) + t * a.heads[0] * a.D;
  T* const yk = static_cast<T*>(a.y[1]) + t * a.heads[1] * a.D;
  for (int u = threadIdx.x; u < units; u += blockDim.x) {
    const bool rot = u < turned;
    // two vectors, one of either half of the values that turn, or of those that pass: lanes side by side in both
    const int at0 = rot ? u * (ADJ && VEC == 1 ? 2 : VEC) : a.rotary + (u - turned) * VEC;
    const int at1 = at0 + (rot ? (ADJ && VEC == 1 ? 1 : a.rotary / 2) : (a.D - a.rotary) / 2);
    float s[VEC], c[VEC];
    if (rot) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int pair = !ADJ || VEC == 1 ? u * VEC + j
                         : j < VEC / 2    ? u * VEC / 2 + j
                                          : a.rotary / 4 + u * VEC / 2 + j - VEC / 2;
        const int ax = min(max(a.axis[pair], 0), a.axes - 1);
        const int64_t at = ax * a.axis_stride + t;
        const int64_t p = a.wide ? static_cast<const int64_t*>(a.positions)[at]
                                 : (int64_t)static_cast<const int32_t*>(a.positions)[at];
        turn((uint64_t)p * a.turns[pair], s[j], c[j]);
        if (a.back) s[j] = -s[j];
      }
    }
    for (int h = h0; h < h1; h += kTogether) {
      P p0[kTogether], p1[kTogether];
#pragma unroll
      for (int i = 0; i < kTogether; ++i) {
        const int g = h + i < h1 ? h + i : h1 - 1;  // the last once more rather than a branch between the loads
        const T* x = g < a.heads[0] ? xq + g * a.head[0] : xk + (g - a.heads[0]) * a.head[1];
        p0[i] = *reinterpret_cast<const P*>(x + at0);
        p1[i] = *reinterpret_cast<const P*>(x + at1);
      }
#pragma unroll
      for (int i = 0; i < kTogether; ++i) {
        const int g = h + i;
        if (g >= h1) break;
        if (rot) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            float l, r;
            if constexpr (!ADJ) {
              l = (float)p0[i][j];
              r = (float)p1[i][j];
              p0[i][j] = (T)(l * c[j] - r * s[j]);
              p1[i][j] = (T)(r * c[j] + l * s[j]);
            } else if constexpr (VEC == 1) {
              l = (float)p0[i][0];
              r = (float)p1[i][0];
              p0[i][0] = (T)(l * c[0] - r * s[0]);
              p1[i][0] = (T)(r * c[0] + l * s[0]);
            } else {
              P& p = 2 * j < VEC ? p0[i] : p1[i];
              l = (float)p[2 * j % VEC];
              r = (float)p[2 * j % VEC + 1];
              p[2 * j % VEC] = (T)(l * c[j] - r * s[j]);
              p[2 * j % VEC + 1] = (T)(r * c[j] + l * s[j]);
            }
          }
        }
        T* y = g < a.heads[0] ? yq + g * a.D : yk + (g - a.heads[0]) * a.D;
        *reinterpret_cast<P*>(y + at0) = p0[i];
        *reinterpret_cast<P*>(y + at1) = p1[i];
      }
    }
  }
}

template <class T, int VEC>
void launch(const RotaryArgs& a, hipStream_t st) {
  const int units = a.D / (2 * VEC), turned = a.rotary / (2 * VEC), heads = a.heads[0] + a.heads[1];
  const int bx = min(units, kThreads), by = kThreads / bx;
  // as many heads a thread as leave 2^18 threads (16 waves a CU)
  int per = min(heads, 16);
  while (per > 1 && a.T * units * ((heads + per - 1) / per) < (1 << 18)) per = (per + 1) / 2;
  const int groups = (heads + per - 1) / per;  // of about one size, whole loads at once
  if (per > kTogether) per = ((heads + groups - 1) / groups + kTogether - 1) / kTogether * kTogether;
  const dim3 grid((unsigned)((a.T + by - 1) / by), (heads + per - 1) / per);
  if (a.adjacent)
    rotary_kernel<T, VEC, true><<<grid, dim3(bx, by), 0, st>>>(a, units, turned, per);
  else
    rotary_kernel<T, VEC, false><<<grid, dim3(bx, by), 0, st>>>(a, units, turned, per);
}

template <class T>
void by_alignment(const RotaryArgs& a, hipStream_t st) {
  constexpr int V = 16 / sizeof(T);
  bool wide = a.D % (2 * V) == 0 && a.rotary % (2 * V) == 0;
  for (int w = 0; w < 2; ++w)
    wide = wide && a.token[w] % V == 0 && a.head[w] % V == 0 && (reinterpret_cast<uintptr_t>(a.x[w]) & 15) == 0 &&
           (reinterpret_cast<uintptr_t>(a.y[w]) & 15) == 0;
  if (wide)
    launch<T, V>(a, st);
  else
    launch<T, 1>(a, st);
}

}  // namespace

void launch_rotary(const RotaryArgs& a, hipStream_t st) {
  if (a.dtype == CQGDN_F32)
    by_alignment<float>(a, st);
  else if (a.dtype == CQGDN_F16)
    by_alignment<_Float16>(a, st);
  else
    by_alignment<__bf16>(a, st);
}

}  // namespace cqgdn
