// The keys' part of the attention's gradients: dv_j = sum_t p_tj dy_t, dk_j = scale sum_t dx_tj q_t (attn_core_bwd.hip has
// the formulas).
//
// A workgroup owns 256 keys, 32 a wave, and goes through the blocks of 64 rows that see any of them, two tiles of Q and dY
// deep.  S = Q K^T and dP = dY V^T: a lane owns a key, and P and dX are already operands of dV^T = dY^T P and dK^T = Q^T dX.
// Two waves a SIMD with 256 registers each: the sums (128 with D = 128) and K stay in them, V's operands come from shared
// memory, as do Q's and dY's.  The exponentials stand between dP's MFMAs and the rest of dX between dV's; what of an MFMA's
// time and of the waits that leaves, the other wave takes.  (One wave a SIMD, with 64 keys and V in registers as well, reads
// half as much from shared memory, but its waits are nobody's: 8192 causal tokens and 1024 queries, 16 heads of 128, 869 us
// where this way took 679.)  That case takes 579 us on a card at full clock, 1100 TFLOP/s of the products that the mask leaves,
// the MFMAs busy for 52% of it; with a cap, three transcendental operations a score, they are for 33%: 13 documents of up to
// 4096 tokens, 16 key heads, 1164 us.
#include <hip/hip_runtime.h>

#include <cstddef>

#include "attn_core_grad.hpp"

namespace cqgdn {
namespace {

// A row's only key has the weight 1 whatever its score: dx is 0, which two orders of the sum dy.v would not leave.  The
// kernel for dq has left such rows' delta as 0 (NaN, where it is not finite), unless lse has a gradient.  `dx`: of the lane's
// key and the rows of the u-th C.
__device__ __forceinline__ void only_keys(const RowBlock& x, int u, int kg, int key, f32x16& dx) {
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int row = c_row(u, e) + 16 * kg;
    if (x.lo[row] == key && x.hi[row] == key + 1) dx[e] = x.delta[row];
  }
}

template <class E, int D>
struct DkvTiles {
  E vt[4][kTileSize<D>], qt[2][kTileSize<D>], yt[2][kTileSize<D>];
  RowBlock info[2];
};
// the workgroup's part of the work, in its shared memory; returns whether it has to be done once more, carefully
template <class E, int D, bool CAP, bool BIAS, bool CAREFUL>
__device__ __forceinline__ bool dkv_keys(const CoreGradArgs& a, int blocks, int splits, DkvTiles<E, D>& tiles) {
  typedef typename Vec<E>::x8 x8;
  constexpr int KQ = D / 16, MT = D / 32;
  static_assert(offsetof(RowBlock, stands) == 1024 && sizeof(RowBlock) == 1536, "an eighth a wave");
  auto& vt = tiles.vt;
  auto& qt = tiles.qt;
  auto& yt = tiles.yt;
  auto& info = tiles.info;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n32 = lane & 31, kg = lane >> 5;
  // the first keys, which most rows see, first
  const int h = blockIdx.x % a.kv_heads, s = blockIdx.x / a.kv_heads % splits;
  const int k0 = blockIdx.x / (a.kv_heads * splits) * kKeys<D>;
  const int group = a.group.d, rows = (int)a.T * group, mine = k0 + 64 * (wave >> 1);
  // the lane's key: as an MFMA takes the rows of a tile
  const int part = wave & 1, key = mine + 16 * (n32 >> 2 & 3) + 8 * part + 4 * (n32 >> 4) + (n32 & 3);
  const TileOperands<E, D> at_tile(lane);
  const Bend bend(a.scale, CAP ? a.cap : 0.f, nullptr, 0);
  // whether a block may have rows of one key: what such a row sees bounds what all see
  const auto may_be_only = [&](const RowRange& x) { return !a.dlse && x.high - x.low <= 1; };

  x8 kf[KQ];  // lane (n32, kg): its key, dimensions 16 i + 8 kg ..
  {
    const bool real = key < a.S;
    const E* k = static_cast<const E*>(a.k) + h * a.k_head + (real ? key : 0) * a.k_token + 8 * kg;
#pragma unroll
    for (int i = 0; i < KQ; ++i)
      kf[i] = __builtin_bit_cast(x8, real ? *reinterpret_cast<const u32x4*>(k + 16 * i) : u32x4{0, 0, 0, 0});
  }
  // the values of all of the workgroup's keys, 32 keys a wave; behind the last key: that key once more
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int block = 2 * wave + i, first = min(k0 + 16 * block, a.S - 1);
    const uint32_t row = min(lane / 4, a.S - 1 - first);
    load_rows16<E, D>(static_cast<const E*>(a.v) + h * a.v_head + first * a.v_token, row * (uint32_t)a.v_token, vt[block / 4], block % 4, lane);
  }
  const E* const vp = vt[wave >> 1];
  f32x16 dk[MT], dv[MT];
  Range<E> range;

  // The blocks of rows, 64 ranges at a time, a lane each: `left` are those of the present 64 that see any of the keys.
  const RowRange* const ranges = static_cast<const RowRange*>(a.ranges);
  int base = -64, turn = s;
  RowRange mine64{};
  uint64_t left = 0;
  const auto next = [&](RowRange& x) -> int {  // the next block of this part, or -1
    while (true) {
      while (left) {
        const int i = __builtin_ctzll(left);
        left &= left - 1;
        if (turn-- == 0) {
          turn = splits - 1;
          x.first = __builtin_amdgcn_readlane(mine64.first, i);
          x.last = __builtin_amdgcn_readlane(mine64.last, i);
          x.low = __builtin_amdgcn_readlane(mine64.low, i);
          x.high = __builtin_amdgcn_readlane(mine64.high, i);
          return base + i;
        }
      }
      base += 64;
      if (base >= blocks) return -1;
      const bool there = base + lane < blocks;
      mine64 = there ? ranges[base + lane] : RowRange{INT32_MAX, 0, 0, 0};
      left = __ballot(there && mine64.last > k0 && mine64.first < k0 + kKeys<D>);
    }
  };
  const auto stage = [&](int block, int buffer) {
    // the first four waves load Q's rows, the others dY's: offsets from the wave's first token; rows behind the last: that
    // once more
    const bool first = wave < 4;
    const int r0 = min(block * kTile + 16 * (wave & 3), rows - 1), t0 = a.group.of(r0);
    const int rho = min(r0 + lane / 4, rows - 1), t = a.group.of(rho), g = rho - t * group;
    const int64_t token = first ? a.q_token : a.dy_token, head = first ? a.q_head : a.dy_head;
    load_rows16<E, D>(static_cast<const E*>(first ? a.q : a.dy) + t0 * token + h * group * head,
                      (t - t0) * (uint32_t)token + g * (uint32_t)head, first ? qt[buffer] : yt[buffer], wave & 3, lane);
    constexpr int size = (BIAS ? sizeof(RowBlock) : offsetof(RowBlock, stands)) / 8;
    const RowBlock* const from = static_cast<const RowBlock*>(a.blocks) + ((int64_t)h * blocks + block);
    if (lane < size / 16)
      load_blocks<1>(reinterpret_cast<const char*>(from) + wave * size, 16 * lane, reinterpret_cast<char*>(&info[buffer]) + wave * size);
  };
  // A step of 64 rows.  WHOLE: all of them see all of the wave's keys.
  const auto step = [&](const E* qp, const E* yp, const RowBlock& x, auto whole, bool only) {
    constexpr bool WHOLE = decltype(whole)::value, APART = CAREFUL && !WHOLE;
    // operands read from LDS ahead of their use, of one and of two an MFMA: as many as leave nothing spilled
    constexpr int kEarly = !WHOLE ? 1 : CAP ? 2 : 3, kEarlyPair = WHOLE && !CAP ? 2 : 1;
    const auto half = [&](int u) {
      f32x16 sc, dp;
      x8 q[KQ], y[KQ], v[KQ];
      const auto query = [&](int i) { q[i] = at_tile.rows(qp, u, i); };
      const auto dy = [&](int i) {
        y[i] = at_tile.rows(yp, u, i);
        v[i] = at_tile.rows(vp, part, i);
      };
      const auto column = [&](const E* p, int i) {
        const x8 c = at_tile.columns(p, u, i / MT, i % MT);
        return APART ? finite_values<E>(c) : c;
      };
      f32x4 lse[4];
      const auto values = [&](const float* p, int i) { return *reinterpret_cast<const f32x4*>(p + c_row(u, 4 * i) + 16 * kg); };
#pragma unroll
      for (int i = 0; i < kEarly; ++i) query(i);
      __builtin_amdgcn_sched_barrier(0);
      sc = f32x16{};
#pragma unroll
      for (int i = 0; i < KQ; ++i) {
        if (i + kEarly < KQ)
          query(i + kEarly);
        else if (i + kEarly - KQ < kEarlyPair)
          dy(i + kEarly - KQ);
        if (i >= KQ - 4) {
          const f32x4 d = values(x.delta, i - KQ + 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) dp[4 * (i - KQ + 4) + e] = d[e];
        }
        if (i == KQ - 1) lse[0] = values(x.lse, 0);
        sc = mfma32(q[i], kf[i], sc);
        __builtin_amdgcn_sched_barrier(0);
      }
      // weights of elements 4 j .. 4 j + 3, from where they are read; with a cap, packed at once, and left times its derivative
      uint32_t pw[8], hidden = 0;
      const auto weights = [&](int j) {
        f32x4 stands, slope;
        u32x4 lo, hi;
        const int row4 = c_row(u, 4 * j) + 16 * kg;
        if constexpr (BIAS) {
          stands = *reinterpret_cast<const f32x4*>(x.stands + row4);
          slope = *reinterpret_cast<const f32x4*>(x.slope + row4);
        }
        if constexpr (!WHOLE) {
          lo = *reinterpret_cast<const u32x4*>(x.lo + row4);
          hi = *reinterpret_cast<const u32x4*>(x.hi + row4);
        }
        f32x4 p, rate;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int e = 4 * j + i;
          if constexpr (!CAP && !BIAS) {
            p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e], bend.c, lse[j][i]));
          } else {
            float r = 1.f, y = lse[j][i];
            if constexpr (CAP)
              y = bend.capped(sc[e], y, r);
            else
              y = __builtin_fmaf(sc[e], bend.c, y);
            if constexpr (BIAS) y = __builtin_fmaf(-slope[i], fabsf(stands[i] - (float)key), y);
            rate[i] = r;
            p[i] = __builtin_amdgcn_exp2f(y);
          }
          if constexpr (!WHOLE) {
            if ((int)(key < (int)lo[i]) | (int)(key >= (int)hi[i])) {
              p[i] = 0.f;
              hidden |= 1u << e;
            }
          }
        }
        if constexpr (CAP) {
          pw[2 * j] = pack2<E>(p[0], p[1]);
          pw[2 * j + 1] = pack2<E>(p[2], p[3]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[4 * j + i] = CAP ? p[i] * rate[i] : p[i];
      };
      x8 yc[2 * MT], qc[2 * MT];
#pragma unroll
      for (int i = 0; i < KQ; ++i) {
        if (i + kEarlyPair < KQ)
          dy(i + kEarlyPair);
        if (i + kEarly >= KQ)
          yc[i + kEarly - KQ] = column(yp, i + kEarly - KQ);
        if (i * 4 % KQ == 0 && i * 4 / KQ < 3) lse[i * 4 / KQ + 1] = values(x.lse, i * 4 / KQ + 1);
        dp = mfma32(y[i], v[i], dp);
#pragma unroll
        for (int j = (i * 4 + KQ - 1) / KQ; j < ((i + 1) * 4 + KQ - 1) / KQ; ++j) weights(j);
        __builtin_amdgcn_sched_barrier(0);
      }
      const auto change = [&](int e) {
        dp[e] *= sc[e];
        if (!WHOLE && (hidden >> e & 1)) dp[e] = 0.f;  // dy may be no finite number there
      };
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = CAP ? pw[4 * b + e] : pack2<E>(sc[8 * b + 2 * e], sc[8 * b + 2 * e + 1]);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const int i = b * MT + m;
          if (i + kEarly < 2 * MT)
            yc[i + kEarly] = column(yp, i + kEarly);
          else
            qc[i + kEarly - 2 * MT] = column(qp, i + kEarly - 2 * MT);
          dv[m] = mfma32(yc[i], __builtin_bit_cast(x8, w), dv[m]);
#pragma unroll
          for (int e = m * 8 / MT; e < (m + 1) * 8 / MT; ++e) change(8 * b + e);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if (!WHOLE && only) only_keys(x, u, kg, key, dp);
      range.fit(dp, dk);
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
          const int i = b * MT + m;
          if (i + kEarly < 2 * MT) qc[i + kEarly] = column(qp, i + kEarly);
          dk[m] = mfma32(qc[i], __builtin_bit_cast(x8, w), dk[m]);
          if constexpr (kTwoTerms<E, WHOLE>) dk[m] = mfma32(qc[i], __builtin_bit_cast(x8, rest), dk[m]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    };
    half(0);
    half(1);
    if (APART && (tile_is_odd<E, D>(qp, lane) || tile_is_odd<E, D>(yp, lane))) {
      const auto sees = [&](int i) { return key >= x.lo[i] && key < x.hi[i]; };
      add_odd<E, D>(qp, dk, lane, sees);
      add_odd<E, D>(yp, dv, lane, sees);
    }
  };

  // the present step's block and range, and the next's, whose tiles are on their way
  RowRange now, later;
  int block, following, buffer;
  const auto ask = [&] {
    following = next(later);
    if (following >= 0) stage(following, buffer ^ 1);
  };
  const auto advance = [&] {
    tiles_ready();
    block = following;
    now = later;
    buffer ^= 1;
  };
#pragma unroll
  for (int i = 0; i < MT; ++i) dk[i] = dv[i] = f32x16{};
  buffer = 0;
  block = next(now);
  if (block >= 0) stage(block, 0);
  tiles_ready();
  // A loop for the whole steps by itself: in one for both kinds, the sums would be moved from the registers that one
  // leaves them in to the other's, in every step.
  while (block >= 0) {
#pragma unroll 1
    while (block >= 0 && now.low <= mine && mine + 64 <= now.high) {
      ask();
      step(qt[buffer], yt[buffer], info[buffer], std::true_type{}, false);
      advance();
    }
    if (block < 0) break;
    ask();
    if (now.last > mine && now.first < mine + 64) step(qt[buffer], yt[buffer], info[buffer], std::false_type{}, may_be_only(now));
    advance();
  }
  if constexpr (!CAREFUL) {
    if (__builtin_amdgcn_readfirstlane(__syncthreads_or(any_not_finite(dk) || any_not_finite(dv)))) return true;
  }
  if (key < a.S) {
    const float f = (CAP ? 4.f : 1.f) * a.scale * range.back() * (Range<E>::on ? 0x1p-15f : 1.f), g = Range<E>::on ? 0x1p-15f : 1.f;
    const int64_t at = ((int64_t)key * a.kv_heads + h) * D, size = (int64_t)a.S * a.kv_heads * D;
    float* const part = a.ws + s * 2 * size;
#pragma unroll
    for (int k = 0; k < MT; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const f32x4 u = f32x4{dk[k][4 * e], dk[k][4 * e + 1], dk[k][4 * e + 2], dk[k][4 * e + 3]} * f;
        const f32x4 w = f32x4{dv[k][4 * e], dv[k][4 * e + 1], dv[k][4 * e + 2], dv[k][4 * e + 3]} * g;
        const int d = 32 * k + 8 * e + 4 * kg;
        if (splits == 1) {
          st4(static_cast<E*>(a.dk) + at + d, u);
          st4(static_cast<E*>(a.dv) + at + d, w);
        } else {
          *reinterpret_cast<f32x4*>(part + at + d) = u;
          *reinterpret_cast<f32x4*>(part + size + at + d) = w;
        }
      }
  }
  return false;
}

// apart from the kernel, whose registers it would cost
template <class E, int D, bool CAP, bool BIAS>
__device__ __noinline__ void dkv_again(CoreGradArgs a, int blocks, int splits, uint32_t tiles) {
  typedef __attribute__((address_space(3))) DkvTiles<E, D>* Tiles;
  dkv_keys<E, D, CAP, BIAS, true>(a, blocks, splits, *(DkvTiles<E, D>*)(Tiles)tiles);
}

template <class E, int D, bool CAP, bool BIAS>
__global__ __launch_bounds__(512, 2) void dkv_kernel(CoreGradArgs a, int blocks, int splits) {
  __shared__ __align__(16) DkvTiles<E, D> tiles;
  if (dkv_keys<E, D, CAP, BIAS, false>(a, blocks, splits, tiles))
    dkv_again<E, D, CAP, BIAS>(a, blocks, splits, (uint32_t)(uintptr_t)(lds_void_ptr)&tiles);
}

// With D = 256 the sums of 32 keys would fill a wave's registers.  Two waves share 32 keys: one forms S, the other dP, they
// exchange them through shared memory, and each sums half of the dimensions; a workgroup takes 64 keys, one wave a SIMD.
// Bound by its waits, and by few workgroups: five documents of up to 1531 tokens with prefixes and slopes, 8 heads, 176 us, in
// which a SIMD has 0.6 waves on average.
template <class E, int D>
struct PairTiles {
  E qt[2][kTileSize<D>], yt[2][kTileSize<D>];
  float swap[4][1024];
  RowBlock info[2];
};
template <class E, int D, bool CAP, bool BIAS, bool CAREFUL>
__device__ __forceinline__ bool pair_keys(const CoreGradArgs& a, int blocks, int splits, PairTiles<E, D>& tiles) {
  typedef typename Vec<E>::x8 x8;
  constexpr int KQ = D / 16, MT = D / 64;
  static_assert(offsetof(RowBlock, stands) == 1024 && sizeof(RowBlock) == 1536, "an instruction, and half of one");
  auto& qt = tiles.qt;
  auto& yt = tiles.yt;
  auto& swap = tiles.swap;
  auto& info = tiles.info;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n32 = lane & 31, kg = lane >> 5;
  const int half = wave & 1;  // of the pair: 0 forms S and sums dimensions below D / 2, 1 dP and those above
  // the first keys, which most rows see, first
  const int h = blockIdx.x % a.kv_heads, s = blockIdx.x / a.kv_heads % splits;
  const int k0 = blockIdx.x / (a.kv_heads * splits) * kKeys<D>;
  const int group = a.group.d, rows = (int)a.T * group, mine = k0 + 32 * (wave >> 1);
  const int key = mine + n32;
  const bool real = key < a.S;
  const TileOperands<E, D> at_tile(lane);
  const Bend bend(a.scale, CAP ? a.cap : 0.f, nullptr, 0);
  // whether a block may have rows of one key: what such a row sees bounds what all see
  const auto may_be_only = [&](const RowRange& x) { return !a.dlse && x.high - x.low <= 1; };

  x8 kf[KQ];  // lane (n32, kg): of key n32 K, in the second wave V, dimensions 16 i + 8 kg ..
  {
    const E* k = static_cast<const E*>(a.k) + h * a.k_head + (real ? key : 0) * a.k_token + 8 * kg;
    const E* v = static_cast<const E*>(a.v) + h * a.v_head + (real ? key : 0) * a.v_token + 8 * kg;
    const u32x4 none{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < KQ; ++i) {
      kf[i] = __builtin_bit_cast(x8, real ? *reinterpret_cast<const u32x4*>((half ? v : k) + 16 * i) : none);
    }
  }
  f32x16 dk[MT], dv[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) dk[i] = dv[i] = f32x16{};
  Range<E> range;

  // The blocks of rows, 64 ranges at a time, a lane each: `left` are those of the present 64 that see any of the keys.
  const RowRange* const ranges = static_cast<const RowRange*>(a.ranges);
  int base = -64, turn = s;
  RowRange mine64{};
  uint64_t left = 0;
  const auto next = [&](RowRange& x) -> int {  // the next block of this part, or -1
    while (true) {
      while (left) {
        const int i = __builtin_ctzll(left);
        left &= left - 1;
        if (turn-- == 0) {
          turn = splits - 1;
          x.first = __builtin_amdgcn_readlane(mine64.first, i);
          x.last = __builtin_amdgcn_readlane(mine64.last, i);
          x.low = __builtin_amdgcn_readlane(mine64.low, i);
          x.high = __builtin_amdgcn_readlane(mine64.high, i);
          return base + i;
        }
      }
      base += 64;
      if (base >= blocks) return -1;
      const bool there = base + lane < blocks;
      mine64 = there ? ranges[base + lane] : RowRange{INT32_MAX, 0, 0, 0};
      left = __ballot(there && mine64.last > k0 && mine64.first < k0 + kKeys<D>);
    }
  };
  const auto stage = [&](int block, int buffer) {
    // offsets from the wave's first token; rows behind the last: that once more
    const int r0 = min(block * kTile + 16 * wave, rows - 1), t0 = a.group.of(r0);
    const int rho = min(r0 + lane / 4, rows - 1), t = a.group.of(rho), g = rho - t * group;
    load_rows16<E, D>(static_cast<const E*>(a.q) + t0 * a.q_token + h * group * a.q_head,
                      (t - t0) * (uint32_t)a.q_token + g * (uint32_t)a.q_head, qt[buffer], wave, lane);
    load_rows16<E, D>(static_cast<const E*>(a.dy) + t0 * a.dy_token + h * group * a.dy_head,
                      (t - t0) * (uint32_t)a.dy_token + g * (uint32_t)a.dy_head, yt[buffer], wave, lane);
    const RowBlock* const from = static_cast<const RowBlock*>(a.blocks) + ((int64_t)h * blocks + block);
    if (wave == 0) load_blocks<1>(from, 16 * lane, &info[buffer]);
    if (BIAS && wave == 1 && lane < 32) load_blocks<1>(from->stands, 16 * lane, info[buffer].stands);
  };
  // of the u-th 32 rows: S or dP - delta
  const auto products = [&](const E* qp, const E* yp, const RowBlock& x, int u, f32x16& sc, f32x16& dp) {
    sc = f32x16{};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4 delta = *reinterpret_cast<const f32x4*>(x.delta + c_row(u, 4 * i) + 16 * kg);
#pragma unroll
      for (int e = 0; e < 4; ++e) dp[4 * i + e] = delta[e];
    }
    if (half) sc = dp;
    const E* const p = half ? yp : qp;
#pragma unroll
    for (int i = 0; i < KQ; ++i) sc = mfma32(at_tile.rows(p, u, i), kf[i], sc);
  };
  const auto give = [&](const f32x16& sc) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<f32x4*>(swap[wave] + 256 * i + 4 * lane) = f32x4{sc[4 * i], sc[4 * i + 1], sc[4 * i + 2], sc[4 * i + 3]};
  };
  const auto take = [&](f32x16& sc, f32x16& dp) {
    f32x16 other;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(swap[wave ^ 1] + 256 * i + 4 * lane);
#pragma unroll
      for (int e = 0; e < 4; ++e) other[4 * i + e] = x[e];
    }
    dp = half ? sc : other;
    sc = half ? other : sc;
  };
  const auto sums = [&](const E* qp, const E* yp, const RowBlock& x, int u, f32x16& sc, f32x16& dp, auto whole,
                        bool only) {
    constexpr bool WHOLE = decltype(whole)::value, APART = CAREFUL && !WHOLE;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row4 = c_row(u, 4 * i) + 16 * kg;
      const f32x4 lse = *reinterpret_cast<const f32x4*>(x.lse + row4);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = 4 * i + j, row = row4 + j;
        float p, rate = 1.f;
        const float from = lse[j];
        p = CAP ? bend.capped(sc[e], from, rate) : __builtin_fmaf(sc[e], bend.c, from);
        if constexpr (BIAS) p = __builtin_fmaf(-x.slope[row], fabsf(x.stands[row] - (float)key), p);
        p = __builtin_amdgcn_exp2f(p);
        float dx = p * dp[e];
        if constexpr (CAP) dx *= rate;
        if constexpr (!WHOLE) {
          const bool hidden = (int)(key < x.lo[row]) | (int)(key >= x.hi[row]);
          if (hidden) p = dx = 0.f;
        }
        sc[e] = p;
        dp[e] = dx;
      }
    }
    if (!WHOLE && only) only_keys(x, u, kg, key, dp);
    range.fit(dp, dk);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      u32x4 w, z, rest;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float one = dp[8 * b + 2 * e] * range.f, two = dp[8 * b + 2 * e + 1] * range.f;
        w[e] = pack2<E>(sc[8 * b + 2 * e], sc[8 * b + 2 * e + 1]);
        z[e] = pack2<E>(one, two);
        if constexpr (kTwoTerms<E, WHOLE>) rest[e] = rest2<E>(one, two, z[e]);
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        x8 y = at_tile.columns(yp, u, b, half * MT + m), q = at_tile.columns(qp, u, b, half * MT + m);
        if constexpr (APART) {
          y = finite_values<E>(y);
          q = finite_values<E>(q);
        }
        dv[m] = mfma32(y, __builtin_bit_cast(x8, w), dv[m]);
        dk[m] = mfma32(q, __builtin_bit_cast(x8, z), dk[m]);
        if constexpr (kTwoTerms<E, WHOLE>) dk[m] = mfma32(q, __builtin_bit_cast(x8, rest), dk[m]);
      }
    }
  };
  const auto step = [&](const E* qp, const E* yp, const RowBlock& x, auto whole, bool only) {
    constexpr bool WHOLE = decltype(whole)::value, APART = CAREFUL && !WHOLE;
    f32x16 sc[2], dp[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) products(qp, yp, x, u, sc[u], dp[u]);
    give(sc[0]);
    lds_barrier();
    take(sc[0], dp[0]);
    lds_barrier();
    give(sc[1]);
    lds_barrier();
    take(sc[1], dp[1]);
#pragma unroll
    for (int u = 0; u < 2; ++u) sums(qp, yp, x, u, sc[u], dp[u], whole, only);
    if (APART && (tile_is_odd<E, D>(qp, lane) || tile_is_odd<E, D>(yp, lane))) {
      const auto sees = [&](int i) { return key >= x.lo[i] && key < x.hi[i]; };
      add_odd<E, D>(qp, dk, lane, sees, half * MT);
      add_odd<E, D>(yp, dv, lane, sees, half * MT);
    }
  };

  RowRange now, later;
  int buffer = 0, block = next(now), following = -1;
  if (block >= 0) stage(block, 0);
  tiles_ready();
  const auto ask = [&] {
    following = next(later);
    if (following >= 0) stage(following, buffer ^ 1);
  };
  const auto advance = [&] {
    tiles_ready();
    block = following;
    now = later;
    buffer ^= 1;
  };
  // The waves meet within a step, so all of them go through every step of the workgroup's, each in its own of the loops.
  while (block >= 0) {
#pragma unroll 1
    while (block >= 0 && now.low <= mine && mine + 32 <= now.high) {
      ask();
      step(qt[buffer], yt[buffer], info[buffer], std::true_type{}, false);
      advance();
    }
    if (block < 0) break;
    ask();
    step(qt[buffer], yt[buffer], info[buffer], std::false_type{}, may_be_only(now));
    advance();
  }
  if constexpr (!CAREFUL) {
    if (__builtin_amdgcn_readfirstlane(__syncthreads_or(any_not_finite(dk) || any_not_finite(dv)))) return true;
  }
  if (real) {
    const float f = (CAP ? 4.f : 1.f) * a.scale * range.back() * (Range<E>::on ? 0x1p-15f : 1.f), g = Range<E>::on ? 0x1p-15f : 1.f;
    const int64_t at = ((int64_t)key * a.kv_heads + h) * D + half * (D / 2);
    float* const part = a.ws + (int64_t)s * 2 * a.S * a.kv_heads * D;
#pragma unroll
    for (int k = 0; k < MT; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const f32x4 u = f32x4{dk[k][4 * e], dk[k][4 * e + 1], dk[k][4 * e + 2], dk[k][4 * e + 3]} * f;
        const f32x4 w = f32x4{dv[k][4 * e], dv[k][4 * e + 1], dv[k][4 * e + 2], dv[k][4 * e + 3]} * g;
        const int d = 32 * k + 8 * e + 4 * kg;
        if (splits == 1) {
          st4(static_cast<E*>(a.dk) + at + d, u);
          st4(static_cast<E*>(a.dv) + at + d, w);
        } else {
          *reinterpret_cast<f32x4*>(part + at + d) = u;
          *reinterpret_cast<f32x4*>(part + (int64_t)a.S * a.kv_heads * D + at + d) = w;
        }
      }
  }
  return false;
}

template <class E, int D, bool CAP, bool BIAS>
__device__ __noinline__ void pair_again(CoreGradArgs a, int blocks, int splits, uint32_t tiles) {
  typedef __attribute__((address_space(3))) PairTiles<E, D>* Tiles;
  pair_keys<E, D, CAP, BIAS, true>(a, blocks, splits, *(PairTiles<E, D>*)(Tiles)tiles);
}

template <class E, int D, bool CAP, bool BIAS>
__global__ __launch_bounds__(256, 1) void pair_kernel(CoreGradArgs a, int blocks, int splits) {
  __shared__ __align__(16) PairTiles<E, D> tiles;
  if (pair_keys<E, D, CAP, BIAS, false>(a, blocks, splits, tiles))
    pair_again<E, D, CAP, BIAS>(a, blocks, splits, (uint32_t)(uintptr_t)(lds_void_ptr)&tiles);
}

}  // namespace

template <class E, int D>
void launch_dkv(const CoreGradArgs& a, int blocks, int splits, hipStream_t st) {
  const unsigned grid = (unsigned)((a.S + kKeys<D> - 1) / kKeys<D> * a.kv_heads * splits);
  by_scores(a, [&](auto cap, auto bias) {
    constexpr bool CAP = decltype(cap)::value, BIAS = decltype(bias)::value;
    if constexpr (D == 256)
      pair_kernel<E, D, CAP, BIAS><<<grid, 256, 0, st>>>(a, blocks, splits);
    else
      dkv_kernel<E, D, CAP, BIAS><<<grid, 512, 0, st>>>(a, blocks, splits);
  });
}
template void launch_dkv<bf16, 64>(const CoreGradArgs&, int, int, hipStream_t);
template void launch_dkv<bf16, 128>(const CoreGradArgs&, int, int, hipStream_t);
template void launch_dkv<bf16, 256>(const CoreGradArgs&, int, int, hipStream_t);
template void launch_dkv<f16, 64>(const CoreGradArgs&, int, int, hipStream_t);
template void launch_dkv<f16, 128>(const CoreGradArgs&, int, int, hipStream_t);
template void launch_dkv<f16, 256>(const CoreGradArgs&, int, int, hipStream_t);

}  // namespace cqgdn
