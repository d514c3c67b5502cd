// New tokens' rows put into the pages of a 16-bit cache, their queries and keys turned by their positions on the way.
//
// As in the rotary kernel a workgroup takes all heads of a few tokens: their sines and cosines are worked out once,
// into LDS, while the first rows are under way; then its threads go through the tokens' heads, queries, keys and
// values, in the order of memory.  Keys and values go to the token's slot in its page, queries to their output, each
// row written once: a token's keys are not written by one launch and read by another.
//
// Bound by memory: 8191 tokens of 16 + 4 + 4 heads of 256 (201 MB read and written) 39 us, 5.1 TB/s.  With two, four and
// eight items' loads of a thread under way at once, and fewer waves a CU for their registers, it was 41, 52 and 63.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "attn_turn.hpp"
#include "cqgdn.h"

namespace cqgdn {
namespace {

constexpr int kThreads = 256;
constexpr int kItems = 4;         // of a thread, one after the other
constexpr int kMostPairs = 4096;  // of a workgroup's tokens: 32 KB of sines and cosines

// The product and sum rounded once, to T.  fp16 has an instruction for it, which the compiler takes in the rotary kernel
// and takes or leaves here, so it is written out (the wait is for a register of which half is written).  (Written out there
// as well, the fp16 rotary kernel takes 2% longer.)
template <class T>
__device__ __forceinline__ T rounded_fma(float a, float b, float c) {
  if constexpr (std::is_same_v<T, _Float16>) {
    uint32_t d;
    asm("v_fma_mixlo_f16 %0, %1, %2, %3\n\ts_nop 1" : "=v"(d) : "v"(a), "v"(b), "v"(c));
    return __builtin_bit_cast(_Float16, (uint16_t)d);
  } else {
    return (T)__builtin_fmaf(a, b, c);
  }
}

// (l c - r s, r c + l s): which product of a sum is rounded first (l s if `left_first`) is not left to the compiler here: it is
// the order that the compiler gives the rotary kernel, as rows appended are that kernel's to the last bit.
template <class T>
__device__ __forceinline__ void turn_pair(T& left, T& right, float s, float c, bool left_first) {
  const float l = (float)left, r = (float)right;
  left = rounded_fma<T>(l, c, -(r * s));
  right = left_first ? rounded_fma<T>(r, c, l * s) : rounded_fma<T>(l, s, r * c);
}

template <class T, int VEC, bool ADJ>
__global__ __launch_bounds__(kThreads) void append_kernel(AppendArgs a, int units, int turned, int tokens, int slots,
                                                             bool left_first) {
  typedef T P __attribute__((ext_vector_type(VEC)));
  typedef TurnPlace<VEC, ADJ> L;
  extern __shared__ __align__(16) float lds[];  // sines [tokens][rotary / 2], then cosines
  const int tid = threadIdx.x, pairs = a.rotary / 2, heads = a.heads[0] + 2 * a.heads[1], size = 1 << a.page_shift;
  const int64_t t0 = (int64_t)blockIdx.x * tokens;
  const int n = (int)min((int64_t)tokens, a.T - t0), items = n * heads;
  float* const sines = lds;
  float* const cosines = lds + tokens * pairs;
  const int slot = tid / units, u = tid - slot * units;
  const L place(a, u, turned);
  const bool working = slot < slots;
  P p0, p1;
  T* y;  // null: not written
  int token;
  bool turns;
  const auto fetch = [&](int item) {
    token = a.by_heads.of(item);
    const int g = item - token * heads, w = g < a.heads[0] ? 0 : g < a.heads[0] + a.heads[1] ? 1 : 2;
    const int h = w == 0 ? g : w == 1 ? g - a.heads[0] : g - a.heads[0] - a.heads[1];
    const int64_t t = t0 + token;
    const T* x = w == 2 ? static_cast<const T*>(a.v) + t * a.v_token + h * a.v_head
                        : static_cast<const T*>(a.x[w]) + t * a.token[w] + h * a.head[w];
    if (w == 0) {
      y = static_cast<T*>(a.y[0]) + (t * a.heads[0] + h) * a.D;
    } else {
      const int at = a.slots[t];
      y = at < 0 || at >= a.slot_count
              ? nullptr
              : static_cast<T*>(a.data) +
                    ((((int64_t)(at >> a.page_shift) * a.heads[1] + h) * 2 + (w - 1)) * size + (at & (size - 1))) * a.D;
    }
    turns = w < 2;
    p0 = *reinterpret_cast<const P*>(x + place.at0);
    p1 = *reinterpret_cast<const P*>(x + place.at1);
  };
  if (working && slot < items) fetch(slot);
  for (int i = tid; i < n * pairs; i += kThreads) {
    const int token = a.by_pairs.of(i);
    angle(a, t0 + token, i - token * pairs, sines[i], cosines[i]);
  }
  __syncthreads();
  if (!working) return;
  for (int item = slot; item < items; item += slots) {
    if (item != slot) fetch(item);
    if (!y) continue;
    if (place.rot && turns) {
#pragma unroll
      for (int j = 0; j < VEC / L::RUN; ++j) {
        const int at = token * pairs + L::pair(a, u, j);
        float s[L::RUN], c[L::RUN];
#pragma unroll
        for (int e = 0; e < L::RUN; ++e) {
          s[e] = sines[at + e];
          c[e] = cosines[at + e];
        }
#pragma unroll
        for (int e = 0; e < L::RUN; ++e) {
          if constexpr (!ADJ || VEC == 1) {
            T l = p0[e], r = p1[e];
            turn_pair(l, r, s[e], c[e], VEC == 1 && left_first);
            p0[e] = l;
            p1[e] = r;
          } else {
            P& p = j ? p1 : p0;
            T l = p[2 * e], r = p[2 * e + 1];
            turn_pair(l, r, s[e], c[e], true);
            p[2 * e] = l;
            p[2 * e + 1] = r;
          }
        }
      }
    }
    *reinterpret_cast<P*>(y + place.at0) = p0;
    *reinterpret_cast<P*>(y + place.at1) = p1;
  }
}

template <class T, int VEC>
void launch(AppendArgs a, bool left_first, hipStream_t st) {
  const int units = a.D / (2 * VEC), turned = a.rotary / (2 * VEC), heads = a.heads[0] + 2 * a.heads[1];
  const int slots = kThreads / units;
  // as many tokens as give a thread kItems, but 1024 workgroups (4 a CU) first
  int64_t tokens = std::max<int64_t>(1, (int64_t)slots * kItems / heads);
  tokens = std::min<int64_t>({tokens, std::max<int64_t>(1, a.T / 1024), std::max(1, kMostPairs / std::max(1, a.rotary / 2))});
  a.by_heads = Divider(heads);
  a.by_pairs = Divider(std::max(1, a.rotary / 2));
  const unsigned grid = (unsigned)((a.T + tokens - 1) / tokens), lds = (unsigned)(tokens * a.rotary * sizeof(float));
  if (a.adjacent)
    append_kernel<T, VEC, true><<<grid, kThreads, lds, st>>>(a, units, turned, (int)tokens, slots, left_first);
  else
    append_kernel<T, VEC, false><<<grid, kThreads, lds, st>>>(a, units, turned, (int)tokens, slots, left_first);
}

template <class T>
void by_alignment(const AppendArgs& a, hipStream_t st) {
  const auto fits = [](int64_t token, int64_t head, const void* p) {
    return token % 8 == 0 && head % 8 == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0;
  };
  const bool turns_wide = a.rotary % 16 == 0 && fits(a.token[0], a.head[0], a.x[0]) && fits(a.token[1], a.head[1], a.x[1]) &&
                          (reinterpret_cast<uintptr_t>(a.y[0]) & 15) == 0;
  const bool left_first = turns_wide && a.adjacent;  // as the rotary kernel's vectors of neighbours
  if (turns_wide && fits(a.v_token, a.v_head, a.v))
    launch<T, 8>(a, left_first, st);
  else
    launch<T, 1>(a, left_first, st);
}

}  // namespace

void launch_append(const AppendArgs& a, hipStream_t st) {
  if (a.dtype == CQGDN_F16)
    by_alignment<_Float16>(a, st);
  else
    by_alignment<__bf16>(a, st);
}

}  // namespace cqgdn
