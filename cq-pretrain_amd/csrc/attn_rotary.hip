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

template <class T, int N>
struct Pack {
  T v[N];
};

// A thread keeps the angles of VEC pairs of one token in registers and takes them through `per` heads,
// so that a sine and cosine (some 40 operations) are paid once for several heads.
template <class T, int VEC, bool ADJ>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a, int units, int turned, int per) {
  const int64_t t = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (t >= a.T) return;
  typedef Pack<T, VEC> P __attribute__((may_alias));
  const int h0 = blockIdx.y * per, h1 = min(h0 + per, a.heads[0] + a.heads[1]);
  for (int u = threadIdx.x; u < units; u += blockDim.x) {
    const bool rot = u < turned;
    float s[VEC], c[VEC];
    int at0, at1;
    if (rot) {
      at0 = ADJ ? u * 2 * VEC : u * VEC;
      at1 = ADJ ? at0 + VEC : a.rotary / 2 + u * VEC;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int pair = u * VEC + j;
        const int ax = min(max(a.axis[pair], 0), a.axes - 1);
        const int64_t at = ax * a.axis_stride + t;
        const int64_t p = a.wide ? static_cast<const int64_t*>(a.positions)[at]
                                 : (int64_t)static_cast<const int32_t*>(a.positions)[at];
        turn((uint64_t)p * a.turns[pair], s[j], c[j]);
        if (a.back) s[j] = -s[j];
      }
    } else {
      at0 = a.rotary + (u - turned) * 2 * VEC;
      at1 = at0 + VEC;
    }
    for (int h = h0; h < h1; ++h) {
      const int w = h >= a.heads[0], g = h - (w ? a.heads[0] : 0);
      const T* x = static_cast<const T*>(a.x[w]) + t * a.token[w] + g * a.head[w];
      T* y = static_cast<T*>(a.y[w]) + (t * a.heads[w] + g) * a.D;
      P p0 = *reinterpret_cast<const P*>(x + at0), p1 = *reinterpret_cast<const P*>(x + at1);
      if (rot) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          T& l = ADJ ? (2 * j < VEC ? p0.v[(2 * j) % VEC] : p1.v[(2 * j) % VEC]) : p0.v[j];
          T& r = ADJ ? (2 * j + 1 < VEC ? p0.v[(2 * j + 1) % VEC] : p1.v[(2 * j + 1) % VEC]) : p1.v[j];
          const float fl = (float)l, fr = (float)r;
          l = (T)(fl * c[j] - fr * s[j]);
          r = (T)(fr * c[j] + fl * s[j]);
        }
      }
      *reinterpret_cast<P*>(y + at0) = p0;
      *reinterpret_cast<P*>(y + at1) = p1;
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
