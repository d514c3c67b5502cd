// Rotary positions with several axes.
//
// A head's first `rotary` values are pairs; pair i turns by the angle position[axis[i]] * f_i, its
// gradient by the opposite angle.  The frequency comes as turns a position in 64-bit fixed point, so
// the low 64 bits of position * turns are the fraction of a turn, exact for every integer position
// (an fp32 product is off by 0.06 rad at position 10^6).  The nearest quarter of a turn leaves its top 32 bits
// and the Taylor polynomials of sine and cosine, degrees 9 and 10 on +-pi/4 (remainders 2e-9 and 1e-10), give
// the rest.
//
// Bound by memory: 32768 tokens of 32 heads of 128 (bf16), forward and backward, 205 us, 5.2 TB/s read and
// written; with the heads of eight tokens side by side in a wave, each eight times 128 bytes, it was 239.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attn_kernels.hpp"
#include "cqgdn.h"

namespace cqgdn {
namespace {

constexpr int kThreads = 256;
constexpr int kTogether = 4;      // items of a thread whose loads are under way at once
constexpr int kMostPairs = 4096;  // of a workgroup's tokens: 32 KB of sines and cosines

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
struct Place {
  int at0, at1;
  bool rot;
  __device__ __forceinline__ Place(const RotaryArgs& a, int u, int turned) : rot(u < turned) {
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

// A workgroup takes all heads of `tokens` tokens.  Their sines and cosines (some 40 operations each) are worked out
// once, into LDS, while the first loads are under way; then its threads go through the tokens' rows in the order
// of memory, kTogether items (a unit of a head) each at once.  `slots` items fit the workgroup.
template <class T, int VEC, bool ADJ>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a, int units, int turned, int tokens, int slots) {
  typedef T P __attribute__((ext_vector_type(VEC)));
  typedef Place<VEC, ADJ> L;
  extern __shared__ __align__(16) float lds[];  // sines [tokens][rotary / 2], then cosines
  const int tid = threadIdx.x, pairs = a.rotary / 2, heads = a.heads[0] + a.heads[1];
  const int64_t t0 = (int64_t)blockIdx.x * tokens;
  const int n = (int)min((int64_t)tokens, a.T - t0), items = n * heads;
  float* const sines = lds;
  float* const cosines = lds + tokens * pairs;
  const int slot = tid / units, u = tid - slot * units;
  const L place(a, u, turned);
  const bool working = slot < slots;
  P p0[kTogether], p1[kTogether];
  T* y[kTogether];
  int token[kTogether];
  const auto fetch = [&](int first) {
#pragma unroll
    for (int i = 0; i < kTogether; ++i) {
      const int item = min(first + i * slots, items - 1);  // the last once more rather than a branch between the loads
      token[i] = a.by_heads.of(item);
      const int g = item - token[i] * heads, w = g >= a.heads[0], h = w ? g - a.heads[0] : g;
      const int64_t t = t0 + token[i];
      const T* x = static_cast<const T*>(a.x[w]) + t * a.token[w] + h * a.head[w];
      y[i] = static_cast<T*>(a.y[w]) + (t * a.heads[w] + h) * a.D;
      p0[i] = *reinterpret_cast<const P*>(x + place.at0);
      p1[i] = *reinterpret_cast<const P*>(x + place.at1);
    }
  };
  if (working) fetch(slot);
  for (int i = tid; i < n * pairs; i += kThreads) {
    const int token = a.by_pairs.of(i);
    angle(a, t0 + token, i - token * pairs, sines[i], cosines[i]);
  }
  __syncthreads();
  if (!working) return;
  for (int first = slot; first < items; first += kTogether * slots) {
    if (first != slot) fetch(first);
#pragma unroll
    for (int i = 0; i < kTogether; ++i) {
      if (first + i * slots >= items) break;
      if (place.rot) {
#pragma unroll
        for (int j = 0; j < VEC / L::RUN; ++j) {
          const int at = token[i] * pairs + L::pair(a, u, j);
          float s[L::RUN], c[L::RUN];
#pragma unroll
          for (int e = 0; e < L::RUN; ++e) {
            s[e] = sines[at + e];
            c[e] = cosines[at + e];
          }
#pragma unroll
          for (int e = 0; e < L::RUN; ++e) {
            if constexpr (!ADJ || VEC == 1) {
              const float l = (float)p0[i][e], r = (float)p1[i][e];
              p0[i][e] = (T)(l * c[e] - r * s[e]);
              p1[i][e] = (T)(r * c[e] + l * s[e]);
            } else {
              P& p = j ? p1[i] : p0[i];
              const float l = (float)p[2 * e], r = (float)p[2 * e + 1];
              p[2 * e] = (T)(l * c[e] - r * s[e]);
              p[2 * e + 1] = (T)(r * c[e] + l * s[e]);
            }
          }
        }
      }
      *reinterpret_cast<P*>(y[i] + place.at0) = p0[i];
      *reinterpret_cast<P*>(y[i] + place.at1) = p1[i];
    }
  }
}

// The same for heads of no vector's size, or too wide for the workgroup: a token a workgroup, a head after the
// other, values by themselves.
template <class T, bool ADJ>
__global__ __launch_bounds__(kThreads) void rotary_any_kernel(RotaryArgs a, int units, int turned) {
  const int64_t t = blockIdx.x;
  for (int u = threadIdx.x; u < units; u += kThreads) {
    const Place<1, ADJ> place(a, u, turned);
    float s = 0.f, c = 1.f;
    if (place.rot) angle(a, t, u, s, c);
    for (int g = 0; g < a.heads[0] + a.heads[1]; ++g) {
      const int w = g >= a.heads[0], h = w ? g - a.heads[0] : g;
      const T* x = static_cast<const T*>(a.x[w]) + t * a.token[w] + h * a.head[w];
      T* y = static_cast<T*>(a.y[w]) + (t * a.heads[w] + h) * a.D;
      T l = x[place.at0], r = x[place.at1];
      if (place.rot) {
        const float fl = (float)l, fr = (float)r;
        l = (T)(fl * c - fr * s);
        r = (T)(fr * c + fl * s);
      }
      y[place.at0] = l;
      y[place.at1] = r;
    }
  }
}

template <class T, int VEC>
void launch(RotaryArgs a, hipStream_t st) {
  const int units = a.D / (2 * VEC), turned = a.rotary / (2 * VEC), heads = a.heads[0] + a.heads[1];
  if (units > kThreads || a.rotary / 2 > kMostPairs) {
    if (a.adjacent)
      rotary_any_kernel<T, true><<<(unsigned)a.T, kThreads, 0, st>>>(a, a.D / 2, a.rotary / 2);
    else
      rotary_any_kernel<T, false><<<(unsigned)a.T, kThreads, 0, st>>>(a, a.D / 2, a.rotary / 2);
    return;
  }
  const int slots = kThreads / units;
  // as many tokens as give a thread two rounds of kTogether items, but 1024 workgroups (4 a CU) first
  int64_t tokens = std::max<int64_t>(1, (int64_t)slots * kTogether * 2 / heads);
  tokens = std::min<int64_t>({tokens, std::max<int64_t>(1, a.T / 1024), std::max(1, kMostPairs / std::max(1, a.rotary / 2))});
  a.by_heads = Divider(heads);
  a.by_pairs = Divider(std::max(1, a.rotary / 2));
  const unsigned grid = (unsigned)((a.T + tokens - 1) / tokens), lds = (unsigned)(tokens * a.rotary * sizeof(float));
  if (a.adjacent)
    rotary_kernel<T, VEC, true><<<grid, kThreads, lds, st>>>(a, units, turned, (int)tokens, slots);
  else
    rotary_kernel<T, VEC, false><<<grid, kThreads, lds, st>>>(a, units, turned, (int)tokens, slots);
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
