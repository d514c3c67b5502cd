// Gradients of the attention over packed rows.
//
// With p the softmax's weights of row t, dy its output's gradient and delta = sum_j p_j dy.v_j (less the gradient of lse):
//   dv_j = sum_t p_tj dy_t,  du_tj = p_tj (dy_t.v_j - delta_t),  dx = du times the cap's derivative,
//   dq_t = scale sum_j dx_tj k_j,  dk_j = scale sum_t dx_tj q_t.
// The weights come again from the scores and the rows' logarithms.  Two kernels, each of which owns what it sums, so
// that nothing is added atomically and results do not depend on timing: one goes through the keys of 128 rows twice, for
// delta and for dq, the other through the rows that see 256 keys for dk and dv, 64 rows a step (attn_core_dkv.hip).  S and dP
// are formed three times, 18 D operations a pair of row and key; a kernel for all, with delta known, would take 10 D.
//
// The first, of which the pass for delta is nearly half, is bound by its phases: MFMAs, exponentials and MFMAs follow each other,
// in the pass for delta behind a wait for each step's keys.  8192 causal tokens and 1024 queries, 16 heads of 128: 812 us,
// the MFMAs busy for 46% of it; 13 documents of up to 4096 tokens, 16 key heads, with a cap: 1559 us, 30%; heads of 256, one
// workgroup a CU: five documents of up to 1531 tokens, 8 heads, 224 us, in which a SIMD has 0.4 waves on average.
//
// The first leaves, for every 64 rows, the range of keys they see, their logarithms and deltas: the second finds its
// steps in those ranges, 64 at a time.  Where its workgroups would not fill the CUs, each takes every n-th of the
// steps, and fp32 parts are added up by a third kernel in their order.
//
// Scores, products, sums are fp32.  p and dx are rounded once to the rows' type for the second products (in bf16 dx to two
// terms where a mask cuts a step).  In fp16, where a dx may be too small or too large for the type, it goes in times a power
// of two that follows the largest so far (of the row, or of the key), and p times 2^15.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "attn_core_grad.hpp"

namespace cqgdn {
namespace {

template <class E, int D>
struct DqTiles {
  E kt[2][kTileSize<D>], vt[2][kTileSize<D>];
};
// the workgroup's part of the work, in its shared memory; returns whether it has to be done once more, carefully
template <class E, int D, bool CAP, bool BIAS, bool CAREFUL>
__device__ __forceinline__ bool dq_rows(const CoreGradArgs& a, int tiles, DqTiles<E, D>& lds) {
  typedef typename Vec<E>::x8 x8;
  constexpr int TOK = kTile, KQ = D / 16, MT = D / 32;
  auto& kt = lds.kt;
  auto& vt = lds.vt;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n32 = lane & 31, kg = lane >> 5;
  // launch order: as the forward pass's
  const int real_blocks = a.kv_heads * tiles;
  int b = blockIdx.x;
  if ((b >> 8 & 1) && (b | 255) < real_blocks) b ^= 255;
  const int tile = tiles - 1 - b / a.kv_heads, h = b % a.kv_heads;
  const int group = a.group.d, T = (int)a.T, rows = T * group;
  const TileOperands<E, D> at_tile(lane);

  const auto limits = [&](int rho, int& lo, int& hi) {
    const int t = a.group.of(rho < rows ? rho : 0);
    lo = rho < rows && a.first ? max(a.first[t], 0) : 0;
    hi = rho < rows ? min(a.visible[t], a.S) : 0;
    if (lo >= hi) lo = hi = 0;
  };
  int first, last;  // the keys that any of the workgroup's rows sees
  {
    int lo0, hi0, lo1, hi1;
    limits(tile * kGradRows + lane, lo0, hi0);
    limits(tile * kGradRows + 64 + lane, lo1, hi1);
    first = min(hi0 > 0 ? lo0 : INT32_MAX, hi1 > 0 ? lo1 : INT32_MAX);
    last = max(hi0, hi1);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      first = min(first, __shfl_xor(first, o, 64));
      last = max(last, __shfl_xor(last, o, 64));
    }
    first = __builtin_amdgcn_readfirstlane(first);
    last = __builtin_amdgcn_readfirstlane(last);
  }
  const int rho = tile * kGradRows + 32 * wave + n32;
  const bool real = rho < rows;
  int lo, hi;
  limits(rho, lo, hi);
  int some = hi > 0 ? lo : INT32_MAX, most = hi, low = lo, high = hi;
#pragma unroll
  for (int i = 1; i < 32; i <<= 1) {
    some = min(some, __shfl_xor(some, i, 64));
    most = max(most, __shfl_xor(most, i, 64));
    low = max(low, __shfl_xor(low, i, 64));
    high = min(high, __shfl_xor(high, i, 64));
  }
  some = __builtin_amdgcn_readfirstlane(some);
  most = __builtin_amdgcn_readfirstlane(most);
  low = __builtin_amdgcn_readfirstlane(low);
  high = __builtin_amdgcn_readfirstlane(high);
  const int block = tile * (kGradRows / kTile) + wave / 2;
  if (h == 0 && (wave & 1) == 0) {  // of 64 rows: a lane each
    int lo1, hi1;
    limits(tile * kGradRows + 32 * wave + lane, lo1, hi1);
    RowRange x{hi1 > 0 ? lo1 : INT32_MAX, hi1, lo1, hi1};
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) {
      x.first = min(x.first, __shfl_xor(x.first, i, 64));
      x.last = max(x.last, __shfl_xor(x.last, i, 64));
      x.low = max(x.low, __shfl_xor(x.low, i, 64));
      x.high = min(x.high, __shfl_xor(x.high, i, 64));
    }
    if (lane == 0) static_cast<RowRange*>(a.ranges)[block] = x;
  }
  const int row_t = real ? a.group.of(rho) : 0, head = h * group + (real ? rho - row_t * group : 0);
  const int64_t at = (int64_t)row_t * a.heads + head;
  const Bend bend(a.scale, CAP ? a.cap : 0.f, BIAS ? a.slopes : nullptr, head);
  const int stands = BIAS && real ? within_reach(a.positions ? a.positions[row_t] : a.visible[row_t] - 1) : 0;

  x8 qf[KQ], yf[KQ];  // lane (n32, kg): q and dy of row n32, dimensions 16 i + 8 kg ..
  {
    const E* q = static_cast<const E*>(a.q) + row_t * a.q_token + head * a.q_head + 8 * kg;
    const E* dy = static_cast<const E*>(a.dy) + row_t * a.dy_token + head * a.dy_head + 8 * kg;
    const u32x4 none{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < KQ; ++i) {
      qf[i] = __builtin_bit_cast(x8, real ? *reinterpret_cast<const u32x4*>(q + 16 * i) : none);
      yf[i] = __builtin_bit_cast(x8, real ? *reinterpret_cast<const u32x4*>(dy + 16 * i) : none);
    }
  }
  const float lse = real ? a.lse[at] * 1.44269504088896341f : 0.f;
  const float base = kWeightBias<E> - lse + bend.cap;
  const auto stage = [&](int j) {
    const int pos = first + j * TOK;
    // rows behind the last key: that key once more
    const uint32_t row = min(16 * wave + lane / 4, a.S - 1 - pos);
    load_rows16<E, D>(static_cast<const E*>(a.k) + h * a.k_head + pos * a.k_token, row * (uint32_t)a.k_token, kt[j & 1], wave, lane);
    load_rows16<E, D>(static_cast<const E*>(a.v) + h * a.v_head + pos * a.v_token, row * (uint32_t)a.v_token, vt[j & 1], wave, lane);
  };
  // delta is formed from the keys and not as dy.out, in which out is rounded: by a delta that is off every dx of the row is
  // off alike, and keys that have something in common (a dimension far from 0) add that up (9216 rows of such keys in bf16:
  // dq off by up to 0.45 times its root mean square with dy.out; in fp16 by an eighth of it).  It costs S and dP once more:
  // forward and backward 1350 -> 1710 us there, in fp16 1500 -> 1870.
  float delta = 0.f;
#pragma unroll 1
  for (int j = 0; first + (int64_t)j * TOK < last; ++j) {
    stage(j);
    tiles_ready();
    const int pos = first + j * TOK;
    if (pos < most && pos + TOK > some) {
      const int lo0 = lo - pos - 16 * kg, hi0 = hi - pos - 16 * kg;
      const float far = BIAS ? (float)(stands - pos - 16 * kg) : 0.f;
#pragma unroll 1
      for (int u = 0; u < 2; ++u) {
        f32x16 sc = f32x16{}, dp = f32x16{};
#pragma unroll
        for (int i = 0; i < KQ; ++i) {
          sc = mfma32(at_tile.rows(kt[j & 1], u, i), qf[i], sc);
          dp = mfma32(at_tile.rows(vt[j & 1], u, i), yf[i], dp);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float x = CAP ? bend.capped(sc[e], bend.cap - lse) : __builtin_fmaf(sc[e], bend.c, -lse);
          if constexpr (BIAS) x = __builtin_fmaf(-bend.slope, fabsf(far - (float)c_row(u, e)), x);
          const int at = c_row(u, e);
          if ((int)(at >= lo0) & (int)(at < hi0)) delta = __builtin_fmaf(__builtin_amdgcn_exp2f(x), dp[e], delta);
        }
      }
    }
    tiles_ready();
  }
  delta += __shfl_xor(delta, 32, 64);
  if (hi - lo == 1 && !a.dlse) {  // dx of an only key is 0: dy.v and delta are one sum, which two orders would not leave 0
    delta *= 0.f;                 // NaN where they are not finite
#pragma unroll
    for (int i = 0; i < KQ; ++i) yf[i] = x8{};
  }
  if (a.dlse && real) delta -= a.dlse[at];
  {
    RowBlock& x = static_cast<RowBlock*>(a.blocks)[(int64_t)h * tiles * (kGradRows / kTile) + block];
    const int n = 32 * (wave & 1) + n32;
    if (kg == 0) {
      x.lse[n] = base;
      x.delta[n] = -delta;
      x.lo[n] = lo;
      x.hi[n] = hi;
      if constexpr (BIAS) {
        x.stands[n] = (float)stands;
        x.slope[n] = bend.slope;
      }
    }
  }

  f32x16 acc[MT];
  Range<E> range;

  const auto step = [&](const E* kp, const E* vp, int pos, auto whole) {
    constexpr bool WHOLE = decltype(whole)::value, APART = CAREFUL && !WHOLE;
    const bool odd = APART && tile_is_odd<E, D>(kp, lane);
    const int lo0 = lo - pos - 16 * kg, hi0 = hi - pos - 16 * kg;
    const float far = (float)(stands - pos - 16 * kg);
    // cut steps one half after the other: a short call's time is that of fetching this code once
#pragma unroll(WHOLE ? 2 : 1)
    for (int u = 0; u < 2; ++u) {
      f32x16 sc = f32x16{}, dp = f32x16{} - delta;
#pragma unroll
      for (int i = 0; i < KQ; ++i) {
        sc = mfma32(at_tile.rows(kp, u, i), qf[i], sc);
        dp = mfma32(at_tile.rows(vp, u, i), yf[i], dp);
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        float x = sc[e], rate = 1.f;
        x = CAP ? bend.capped(x, base, rate) : __builtin_fmaf(x, bend.c, base);
        if constexpr (BIAS) x = __builtin_fmaf(-bend.slope, fabsf(far - (float)c_row(u, e)), x);
        x = __builtin_amdgcn_exp2f(x) * dp[e];
        if constexpr (CAP) x *= rate;
        const int at = c_row(u, e);
        if (!WHOLE && ((int)(at < lo0) | (int)(at >= hi0))) x = 0.f;
        dp[e] = x;
      }
      range.fit(dp, acc);
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        u32x4 w, rest;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = dp[8 * b + 2 * e] * range.f, y = dp[8 * b + 2 * e + 1] * range.f;
          w[e] = pack2<E>(x, y);
          if constexpr (kTwoTerms<E, WHOLE>) rest[e] = rest2<E>(x, y, w[e]);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          x8 k = at_tile.columns(kp, u, b, m);
          if (APART) k = finite_values<E>(k);
          acc[m] = mfma32(k, __builtin_bit_cast(x8, w), acc[m]);
          if constexpr (kTwoTerms<E, WHOLE>) acc[m] = mfma32(k, __builtin_bit_cast(x8, rest), acc[m]);
        }
      }
    }
    if (odd) add_odd<E, D>(kp, acc, lane, [&](int i) { return pos + i >= lo && pos + i < hi; });
  };

  const int n = last > 0 ? (last - first + TOK - 1) / TOK : 0;
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = f32x16{};
  if (n > 0) {
    stage(0);
    tiles_ready();
  }
  int j = 0, pos = first;
  const auto advance = [&] {
    tiles_ready();
    ++j;
    pos += TOK;
  };
  // A loop for the whole steps by itself: in one for both kinds, the sums would be moved from the registers that one
  // leaves them in to the other's, in every step.
  while (j < n) {
#pragma unroll 1
    while (j < n && pos >= low && pos + TOK <= high) {
      if (j + 1 < n) stage(j + 1);
      step(kt[j & 1], vt[j & 1], pos, std::true_type{});
      advance();
    }
    if (j == n) break;
    if (j + 1 < n) stage(j + 1);
    if (pos < most && pos + TOK > some) step(kt[j & 1], vt[j & 1], pos, std::false_type{});
    advance();
  }
  if constexpr (!CAREFUL) {
    if (__builtin_amdgcn_readfirstlane(__syncthreads_or(any_not_finite(acc)))) return true;
  }
  if (real) {
    const float f = (CAP ? 4.f : 1.f) * a.scale * range.back() * (Range<E>::on ? 0x1p-15f : 1.f);
#pragma unroll
    for (int k = 0; k < MT; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        st4(static_cast<E*>(a.dq) + at * D + 32 * k + 8 * e + 4 * kg,
            f32x4{acc[k][4 * e], acc[k][4 * e + 1], acc[k][4 * e + 2], acc[k][4 * e + 3]} * f);
  }
  return false;
}

// apart from the kernel, whose registers it would cost
template <class E, int D, bool CAP, bool BIAS>
__device__ __noinline__ void dq_again(CoreGradArgs a, int tiles, uint32_t lds) {
  typedef __attribute__((address_space(3))) DqTiles<E, D>* Tiles;
  dq_rows<E, D, CAP, BIAS, true>(a, tiles, *(DqTiles<E, D>*)(Tiles)lds);
}

template <class E, int D, bool CAP, bool BIAS>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void dq_kernel(CoreGradArgs a, int tiles) {
  __shared__ __align__(16) DqTiles<E, D> lds;
  if (dq_rows<E, D, CAP, BIAS, false>(a, tiles, lds))
    dq_again<E, D, CAP, BIAS>(a, tiles, (uint32_t)(uintptr_t)(lds_void_ptr)&lds);
}

// the parts of dk and dv, added up in their order, 4 values a thread
template <class E>
__global__ __launch_bounds__(256) void join_parts_kernel(const float* ws, int64_t size, int splits, E* dk, E* dv) {
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= 2 * size) return;
  f32x4 y = *reinterpret_cast<const f32x4*>(ws + at);
#pragma unroll 4
  for (int s = 1; s < splits; ++s) y += *reinterpret_cast<const f32x4*>(ws + s * 2 * size + at);
  st4(at < size ? dk + at : dv + (at - size), y);
}

// blocks of 64 rows, of whole workgroups for dq
int64_t row_blocks(int64_t T, int group) { return (T * group + kGradRows - 1) / kGradRows * (kGradRows / kTile); }

// Parts of the keys' gradients: no more than give two rounds of workgroups, one a CU, and no more than pay.  A step of 64
// rows takes a workgroup that is alone some 2.5 us, a part's fp32 sums 16 bytes a value, written and read: b blocks of rows
// over n parts 2.5 b / n + 3.3e-6 n S kv_heads D us, which is least at sqrt(750000 b / (S kv_heads D)) parts (2304 rows:
// 10 parts 92 us with the join, 16 111; 317 rows: 30 either way).
int key_parts(int64_t T, int64_t S, int kv_heads, int group, int D) {
  const int keys = D == 256 ? kKeys<256> : D == 128 ? kKeys<128> : kKeys<64>;
  const int64_t each = std::max<int64_t>(1, (S + keys - 1) / keys * kv_heads), blocks = row_blocks(T, group);
  const int64_t pays = (int64_t)std::lround(std::sqrt(750000. * blocks / std::max<int64_t>(1, S * kv_heads * D)));
  return (int)std::max<int64_t>(1, std::min<int64_t>({512 / each, 16, blocks, pays}));
}

template <class E, int D>
void launch_grad(const CoreGradArgs& a, hipStream_t st) {
  const int group = a.heads / a.kv_heads, tiles = (int)(row_blocks(a.T, group) / (kGradRows / kTile));
  const int splits = key_parts(a.T, a.S, a.kv_heads, group, D);
  if (tiles > 0)
    by_scores(a, [&](auto cap, auto bias) {
      dq_kernel<E, D, decltype(cap)::value, decltype(bias)::value><<<tiles * a.kv_heads, 256, 0, st>>>(a, tiles);
    });
  if (a.S == 0 || !a.dk) return;
  launch_dkv<E, D>(a, tiles * (kGradRows / kTile), splits, st);
  if (splits > 1) {
    const int64_t size = (int64_t)a.S * a.kv_heads * D;
    join_parts_kernel<E><<<(unsigned)((2 * size + 1023) / 1024), 256, 0, st>>>(a.ws, size, splits, static_cast<E*>(a.dk), static_cast<E*>(a.dv));
  }
}

template <class E>
void by_dim(const CoreGradArgs& a, hipStream_t st) {
  if (a.D == 64)
    launch_grad<E, 64>(a, st);
  else if (a.D == 128)
    launch_grad<E, 128>(a, st);
  else
    launch_grad<E, 256>(a, st);
}

}  // namespace

// the row blocks, their ranges, and the parts where there are several
static size_t backward_layout(int64_t T, int64_t S, int heads, int kv_heads, int D, size_t& ranges, size_t& parts) {
  const int group = heads / kv_heads;
  const int64_t blocks = row_blocks(T, group);
  const int splits = key_parts(T, S, kv_heads, group, D);
  ranges = (size_t)blocks * kv_heads * sizeof(RowBlock);
  parts = ((ranges + blocks * sizeof(RowRange)) + 255) / 256 * 256;
  return parts + (splits > 1 ? (size_t)splits * 2 * S * kv_heads * D * sizeof(float) : 0);
}
size_t core_backward_bytes(int64_t T, int64_t S, int heads, int kv_heads, int D) {
  size_t ranges, parts;
  return backward_layout(T, S, heads, kv_heads, D, ranges, parts);
}

void launch_core_backward(const CoreGradArgs& args, hipStream_t st) {
  CoreGradArgs a = args;
  size_t ranges, parts;
  backward_layout(a.T, a.S, a.heads, a.kv_heads, a.D, ranges, parts);
  char* const ws = reinterpret_cast<char*>(args.ws);
  a.blocks = ws;
  a.ranges = ws + ranges;
  a.ws = reinterpret_cast<float*>(ws + parts);
  if (a.fp16)
    by_dim<f16>(a, st);
  else
    by_dim<bf16>(a, st);
}

}  // namespace cqgdn
