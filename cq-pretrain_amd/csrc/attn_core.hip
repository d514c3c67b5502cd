// Attention over 16-bit keys and values, many rows: packed documents in training, prompts over a paged cache.
//
// Row (t, query head) gets sum_j p_j v_j / sum_j p_j over the keys j that it sees, p_j = exp(u_j - m), u_j its capped
// and biased score, in one pass with a running maximum m.  A workgroup takes 128 rows of one key head, 32 a wave (with
// grouped heads a row is a token and one of the group's query heads, so that the group shares K and V), and 64
// keys a step, whose K and V rows go from memory to shared memory without passing registers, two steps deep.  S^T =
// K Q^T and O^T = V^T P^T: a lane owns a row, so limits, maximum, sum and the head's slope are the lane's own and S^T's
// layout is already an operand of O^T.  Steps that all of a wave's rows see whole, most of them, have no masks.
//
// Bound by the MFMAs and, at about as many cycles, the operations on scores that stand between them: 8192 causal tokens and
// 1024 queries, 16 heads of 128, 326 us, 975 TFLOP/s of the products that the mask leaves; the MFMAs are busy for half of it.
// With a cap they are for 28%, and the VALU for 37% at four cycles an operation (its transcendental ones take more): neither
// is full, as the cap's exponentials and reciprocals stand alone between the groups of MFMAs (13 documents of up to 4096
// tokens, 16 key heads: 654 us).  With heads of 64 a score has half the MFMA work: 21% and 48% (seven documents with a window
// of 1024: 97 us).
//
// Scores, sums and O are fp32; a weight is rounded once to the rows' type for its product with V (half a step of
// the type times sum p |v| / sum p in a result).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attn_core.hpp"
#include "attn_plan.hpp"

namespace cqgdn {
namespace {

constexpr int kRows = 128;  // of a workgroup, 32 a wave

// which rows a workgroup takes: request r's (from `from` on, `rows` with the group's heads) of key head h, tile after tile
struct CorePlace {
  int h, r, s, splits, from, rows;
  bool padding;
};
template <class E, int D>
struct CoreTiles {
  E kt[2][kTileSize<D>], vt[2][kTileSize<D>];
};
// One tile of 128 rows, in the workgroup's shared memory.
// PAGED: keys from the pages of a cache; CAP, BIAS: scores are capped, biased
template <class E, int D, bool PAGED, bool CAP, bool BIAS>
__device__ __forceinline__ void core_tile(const CoreArgs& a, const CorePlace place, int tile, CoreTiles<E, D>& lds) {
  typedef typename Vec<E>::x8 x8;
  constexpr int TOK = kTile, KQ = D / 16, MT = D / 32;
  constexpr int F = 2 * KQ, H = 2 * MT;  // operands of a step: K's, and V's for 32 keys
  // operands read from LDS ahead of their MFMA: K's, and V's while the scores of the second 32 keys are formed
  constexpr int kEarly = 8, kFirst = H < 8 ? H : 8;
  constexpr int GROUPS = TOK / 16;
  auto& kt = lds.kt;
  auto& vt = lds.vt;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n32 = lane & 31, kg = lane >> 5;
  const int h = place.h, r = place.r, s = place.s, splits = place.splits, from = place.from, rows = place.rows;
  const bool padding = place.padding;
  const int requests = PAGED ? a.N : 1, group = a.group.d, size = 1 << a.page_shift;
  const int room = PAGED ? (int)min((int64_t)a.columns << a.page_shift, (int64_t)kAttendRoom) : a.S;
  // A score is c times what is held of it, plus `above`, less the bias.  Held is q.k (the factor is never 0, so that a masked
  // score stays -infinity; its sign goes with Q) or, of a capped score, -r.
  const float c = CAP ? 2.f * a.cap * 1.44269504088896341f : fmaxf(fabsf(a.scale) * 1.44269504088896341f, 1.17549435e-38f);
  const float above = CAP ? a.cap * 1.44269504088896341f : 0.f;
  constexpr float bias = kAttendBias<E>;
  const TileOperands<E, D> at_tile(lane);

  const auto limits = [&](int rho, int& lo, int& hi) {
    const int t = from + a.group.of(rho < rows ? rho : 0);
    if constexpr (PAGED) {
      attend_limits(rho < rows && r < a.N ? a.visible[t] : 0, a.window, room, lo, hi);
    } else {
      lo = rho < rows && a.first ? max(a.first[t], 0) : 0;
      hi = rho < rows ? min(a.visible[t], room) : 0;
      if (lo >= hi) lo = hi = 0;
    }
  };
  // what the workgroup's rows see together
  int first, last;
  {
    int lo0, hi0, lo1, hi1;
    limits(tile * kRows + lane, lo0, hi0);
    limits(tile * kRows + 64 + lane, lo1, hi1);
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
  const int rho = tile * kRows + 32 * wave + n32;
  const bool real = rho < rows;
  int lo, hi;
  limits(rho, lo, hi);
  // what any of the wave's rows sees, and what all of them see, where nothing is masked
  int some = hi > 0 ? lo : INT32_MAX, most = hi, low = lo, high = real ? hi : INT32_MAX;
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
  const int row_t = real ? a.group.of(rho) : 0, t = from + row_t, head = h * group + (real ? rho - row_t * group : 0);
  x8 qf[KQ];  // lane (n32, kg): row n32, dimensions 16 i + 8 kg ..
  {
    const E* q = static_cast<const E*>(a.q) + t * a.q_token + head * a.q_head + 8 * kg;
#pragma unroll
    for (int i = 0; i < KQ; ++i) {
      u32x4 w = real ? *reinterpret_cast<const u32x4*>(q + 16 * i) : u32x4{0, 0, 0, 0};
      if (!CAP && a.scale < 0.f) w ^= 0x80008000u;
      qf[i] = __builtin_bit_cast(x8, w);
    }
  }
  const Bend bend(a.scale, CAP ? a.cap : 0.f, BIAS ? a.slopes : nullptr, head);
  int stands = BIAS && real && r < requests ? (a.positions ? a.positions[t] : a.visible[t] - 1) : 0;
  if (!PAGED) stands = within_reach(stands);
  f32x16 o[MT];
  float m, l;

  const int begin = last > 0 ? (PAGED ? first & ~(TOK - 1) : first) : 0;
  const int steps = (last - begin + TOK - 1) / TOK, per = (steps + splits - 1) / splits;
  const int n = min(steps, (s + 1) * per) - s * per;
  // Steps go from the first key to the last; with a bias, which is least at a row's own position, the other way, so that a
  // row's maximum is found early (steep slopes had it move in every step: seven documents with a window of 1024, heads of
  // 64, 154 us, this way 106)
  const int pos0 = begin + (s * per + (BIAS ? n - 1 : 0)) * TOK;
  constexpr int FURTHER = BIAS ? -TOK : TOK;

  // the block table's entries for the 16 positions each of step j, one a lane
  const auto entries = [&](int j) {
    const int column = (pos0 + j * FURTHER + 16 * (lane & (GROUPS - 1))) >> a.page_shift;
    return j < n && column < a.columns ? a.tables[r * a.table_stride + column] : -1;
  };
  // step j's rows of the wave on their way into the tiles.  Returns which of the step's 16 positions are shown.
  const auto stage = [&](int table, int j) {
    const int pos = pos0 + j * FURTHER;
    if constexpr (PAGED) {
      const uint32_t page = __builtin_amdgcn_readlane(table, wave);
      const int at = (pos + 16 * wave) & (size - 1);
      const E* base = reinterpret_cast<const E*>(a.data) +
                      (((int64_t)(page < a.page_count ? page : 0) * a.kv_heads + h) * 2 * size + at) * D;
      load_rows16<E, D>(base, lane / 4 * D, kt[j & 1], wave, lane);
      load_rows16<E, D>(base + size * D, lane / 4 * D, vt[j & 1], wave, lane);
      return (int)__ballot((uint32_t)table < a.page_count) & ((1 << GROUPS) - 1);
    } else {
      // rows behind the last key: that key once more
      const uint32_t row = min(16 * wave + lane / 4, a.S - 1 - pos);
      load_rows16<E, D>(static_cast<const E*>(a.k) + h * a.k_head + pos * a.k_token, row * (uint32_t)a.k_token, kt[j & 1], wave, lane);
      load_rows16<E, D>(static_cast<const E*>(a.v) + h * a.v_head + pos * a.v_token, row * (uint32_t)a.v_token, vt[j & 1], wave, lane);
      return (1 << GROUPS) - 1;
    }
  };
  // the weights of 32 keys, two a part, in the order of their scores
  float base, sum;
  const auto begin_weights = [&]() {
    base = above + bias - (m == -INFINITY ? 0.f : m);
    sum = 0.f;
  };
  // of element e of the u-th scores of a step `far` from the row, with `more`
  const auto scored = [&](const f32x16& s, int u, float far, int e, float more) {
    if constexpr (BIAS) more = __builtin_fmaf(-bend.slope, fabsf(far - (float)c_row(u, e)), more);
    return __builtin_fmaf(s[e], c, more);
  };
  const auto weights = [&](const f32x16& s, uint32_t (&w)[8], int u, float far, int i) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef E x2 __attribute__((ext_vector_type(2)));
    f32x2 p;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      p[e] = __builtin_amdgcn_exp2f(scored(s, u, far, 2 * i + e, base));
      sum += p[e];
    }
    w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(p, x2));
  };
  const auto capped = [&](f32x16& s) {
    if constexpr (CAP) {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = bend.less_r(s[e]);
    }
  };
  // where the weights have grown too large, or are a row's first, its maximum moves and they are made again
  const auto settle = [&](const f32x16& s, uint32_t (&w)[8], int u, float far) {
    bool large = sum > kAttendLimit<E> || m == -INFINITY;
    if (__any(large)) {
      large = __shfl_xor((int)large, 32, 64) || large;  // the two lanes of a row
      float top = scored(s, u, far, 0, above);
#pragma unroll
      for (int e = 1; e < 16; ++e) top = fmaxf(top, scored(s, u, far, e, above));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      if (large && top > m) {
        const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
        m = top;
        l *= f;
#pragma unroll
        for (int k = 0; k < MT; ++k) o[k] *= f;
      }
      begin_weights();
#pragma unroll
      for (int i = 0; i < 8; ++i) weights(s, w, u, far, i);
    }
    l += sum;
  };
  const auto weight8 = [&](const uint32_t (&w)[8], int i) {
    return __builtin_bit_cast(x8, u32x4{w[i], w[i + 1], w[i + 2], w[i + 3]});
  };
  // a step that all of the wave's rows see whole
  const auto whole_step = [&](const E* kp, const E* vp, int pos) {
    x8 kf[F], vf[2][H];
    f32x16 sc[2];
    uint32_t pw[2][8];
    const float far = (float)__builtin_elementwise_sub_sat(stands, pos + 16 * kg);
    const auto key = [&](int i) { kf[i] = at_tile.rows(kp, i / KQ, i % KQ); };
    const auto value = [&](int u, int i) { vf[u][i] = at_tile.columns(vp, u, i / MT, i % MT); };
#pragma unroll
    for (int i = 0; i < kEarly && i < F; ++i) key(i);
    const auto score = [&](int u, int i) {
      if (i == 0) sc[u] = f32x16{};
      sc[u] = mfma32(kf[u * KQ + i], qf[i], sc[u]);
      if (u * KQ + i + kEarly < F) key(u * KQ + i + kEarly);
    };
    const auto gather = [&](int u, int i) { o[i % MT] = mfma32(vf[u][i], weight8(pw[u], i / MT * 4), o[i % MT]); };
    // An MFMA leaves the wave's issue free for about as long as two weights take.  So the first 32 keys' weights
    // stand between the second's scores, the second's between the first's products with V.
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < KQ; ++i) {
      score(0, i);
      __builtin_amdgcn_sched_barrier(0);
    }
    capped(sc[0]);
    begin_weights();
#pragma unroll
    for (int i = 0; i < KQ; ++i) {
      score(1, i);
#pragma unroll
      for (int e = i * 8 / KQ; e < (i + 1) * 8 / KQ; ++e) weights(sc[0], pw[0], 0, far, e);
#pragma unroll
      for (int e = i * kFirst / KQ; e < (i + 1) * kFirst / KQ; ++e) value(0, e);
      __builtin_amdgcn_sched_barrier(0);
    }
    settle(sc[0], pw[0], 0, far);
    capped(sc[1]);
    begin_weights();
#pragma unroll
    for (int i = 0; i < H; ++i) {
      gather(0, i);
#pragma unroll
      for (int e = i * 8 / H; e < (i + 1) * 8 / H; ++e) weights(sc[1], pw[1], 1, far, e);
      if (i + kFirst < H)
        value(0, i + kFirst);
      else
        value(1, i + kFirst - H);
      __builtin_amdgcn_sched_barrier(0);
    }
    settle(sc[1], pw[1], 1, far);
#pragma unroll
    for (int i = 0; i < H; ++i) {
      gather(1, i);
      if (i + kFirst < H) value(1, i + kFirst);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // one that they do not: hidden keys leave the scores, and values that are not finite reach only rows that see them
  const auto cut_step = [&](const E* kp, const E* vp, int pos, int shown, auto careful) {
    constexpr bool CAREFUL = decltype(careful)::value;
    const int lo0 = lo - pos - 16 * kg, hi0 = hi - pos - 16 * kg;
    const float far = (float)__builtin_elementwise_sub_sat(stands, pos + 16 * kg);
    const bool odd = CAREFUL && tile_is_odd<E, D>(vp, lane);
    // one half after the other: a short call's time is that of fetching this code once
#pragma unroll 1
    for (int u = 0; u < 2; ++u) {
      f32x16 sc = f32x16{};
      uint32_t pw[8];
#pragma unroll
      for (int i = 0; i < KQ; ++i) sc = mfma32(at_tile.rows(kp, u, i), qf[i], sc);
      capped(sc);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int at = c_row(u, e);
        if ((int)(at < lo0) | (int)(at >= hi0) | (int)!(shown >> (2 * (e >> 2 & 1) + kg) & 1)) sc[e] = -INFINITY;
      }
      begin_weights();
#pragma unroll
      for (int e = 0; e < 8; ++e) weights(sc, pw, u, far, e);
      settle(sc, pw, u, far);
#pragma unroll
      for (int i = 0; i < H; ++i) {
        x8 v = at_tile.columns(vp, u, i / MT, i % MT);
        if (odd) v = finite_values<E>(v);
        o[i % MT] = mfma32(v, weight8(pw, i / MT * 4), o[i % MT]);
      }
    }
    if (odd)
      add_odd<E, D>(vp, o, lane, [&](int i) { return pos + i >= lo && pos + i < hi && (shown >> (i >> 4) & 1); });
  };

  for (bool careful = false;;) {
#pragma unroll
    for (int i = 0; i < MT; ++i) o[i] = f32x16{};
    m = hi > 0 ? -INFINITY : 0.f;
    l = 0.f;
    if (n <= 0) break;
    int table1 = -1, shown1 = 0, j = 0, pos = pos0;
    if constexpr (PAGED) table1 = entries(1);
    int shown = stage(PAGED ? entries(0) : -1, 0);
    tiles_ready();
    const auto ask = [&] {
      if (j + 1 < n) shown1 = stage(table1, j + 1);
      if constexpr (PAGED) table1 = entries(j + 2);
    };
    const auto advance = [&] {
      tiles_ready();
      shown = shown1;
      ++j;
      pos += FURTHER;
    };
    // A loop for the whole steps by itself: in one for both kinds, the sums would be moved from the registers that one
    // leaves them in to the other's, in every step.
    while (j < n) {
#pragma unroll 1
      while (j < n && pos >= low && pos + TOK <= high && shown == (1 << GROUPS) - 1) {
        ask();
        whole_step(kt[j & 1], vt[j & 1], pos);
        advance();
      }
      if (j == n) break;
      ask();
      if (pos < most && pos + TOK > some) {
        if (careful)
          cut_step(kt[j & 1], vt[j & 1], pos, shown, std::true_type{});
        else
          cut_step(kt[j & 1], vt[j & 1], pos, shown, std::false_type{});
      }
      advance();
    }
    if (careful || !__builtin_amdgcn_readfirstlane(__syncthreads_or(any_not_finite(o)))) break;
    careful = true;
  }
  l += __shfl_xor(l, 32, 64);
  // No weight above 0: the row's keys are hidden here, or the scores of all are -infinity.
  if (l == 0.f && hi > 0 && n > 0) {
    const int from_key = max(lo, begin + s * per * TOK), to_key = min(hi, begin + min(steps, (s + 1) * per) * TOK);
    if (PAGED ? pages_hold(a, r, from_key, to_key) : from_key < to_key) l = splits > 1 ? kNoWeight : __builtin_nanf("");
  }
  if (real) {
    const int64_t at = (int64_t)t * a.heads + head;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (splits == 1 || l != 0.f) {  // the join reads no part that saw nothing
#pragma unroll
      for (int k = 0; k < MT; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f32x4 y{o[k][4 * e], o[k][4 * e + 1], o[k][4 * e + 2], o[k][4 * e + 3]};
          const int d = 32 * k + 8 * e + 4 * kg;
          if (splits == 1)
            st4(static_cast<E*>(a.out) + at * D + d, l == 0.f ? zero4() : y * inv);
          else
            *reinterpret_cast<f32x4*>(a.ws + (at * splits + s) * D + d) = y;
        }
    }
    if (kg == 0) {
      if (splits > 1) {
        for (int part = s; part < (padding ? splits : s + 1); ++part) {
          float* ml = a.ws + a.T * a.heads * splits * D + (at * splits + part) * 2;
          ml[0] = l == 0.f ? -INFINITY : m;
          ml[1] = l;
        }
      } else if (a.lse) {
        a.lse[at] = (m - bias + log2f(l)) * 0.693147180559945309f;
      }
    }
  }
}

template <class E, int D, bool PAGED, bool CAP, bool BIAS>
__global__ __launch_bounds__(256, D == 256 ? 1 : D == 64 ? 3 : 2) void core_kernel(CoreArgs a, int tiles, int splits) {
  __shared__ __align__(16) CoreTiles<E, D> lds;
  // Launch order: the last tiles, which see most, first; every other round of 256 workgroups reversed, so that
  // a CU's workgroups add up to the same.  Rows behind the requests' ("request N") come last.
  const int requests = PAGED ? a.N : 1, each = a.kv_heads * requests * splits, real_blocks = each * tiles;
  int b = blockIdx.x;
  const bool padding = PAGED && b >= real_blocks;
  if (padding)
    b -= real_blocks;
  else if ((b >> 8 & 1) && (b | 255) < real_blocks)
    b ^= 255;
  const int heads_each = padding ? a.kv_heads : each;
  const int tile0 = padding ? b / heads_each : tiles - 1 - b / heads_each;
  b %= heads_each;
  const int s = padding ? 0 : b % splits;
  if (!padding) b /= splits;
  const int h = b % a.kv_heads, r = padding ? a.N : b / a.kv_heads;
  if (padding) tiles = (gridDim.x - real_blocks) / a.kv_heads;
  const int T = (int)a.T;
  int from = 0, to = T;
  if constexpr (PAGED) {
    from = r == 0 ? 0 : min(max(a.starts[r], 0), T);
    to = padding ? T : min(max(a.starts[r + 1], from), T);
  }
  const CorePlace place{h, r, s, splits, from, (to - from) * (int)a.group.d, padding};
  for (int tile = tile0; tile * kRows < place.rows; tile += tiles) core_tile<E, D, PAGED, CAP, BIAS>(a, place, tile, lds);
}

template <class E, int D, bool PAGED>
void launch(const CoreArgs& a, int splits, hipStream_t st) {
  const int64_t requests = PAGED ? a.N : 1, each = std::max<int64_t>(1, requests * a.kv_heads * splits);
  const int64_t wanted = ((int64_t)(PAGED ? a.max_queries : a.T) * (a.heads / a.kv_heads) + kRows - 1) / kRows;
  const int tiles = (int)std::max<int64_t>(1, std::min<int64_t>(wanted, (1 << 23) / each));
  const int64_t blocks = requests * a.kv_heads * splits * tiles + (PAGED ? (int64_t)a.kv_heads * std::min(tiles, 16) : 0);
  by_scores(a, [&](auto cap, auto bias) {
    core_kernel<E, D, PAGED, decltype(cap)::value, decltype(bias)::value><<<(unsigned)blocks, 256, 0, st>>>(a, tiles, splits);
  });
}

template <class E, int D>
void by_kind(const CoreArgs& a, bool paged, int splits, hipStream_t st) {
  paged ? launch<E, D, true>(a, splits, st) : launch<E, D, false>(a, splits, st);
}

template <class E>
void by_dim(const CoreArgs& a, bool paged, int splits, hipStream_t st) {
  if (a.D == 64)
    by_kind<E, 64>(a, paged, splits, st);
  else if (a.D == 128)
    by_kind<E, 128>(a, paged, splits, st);
  else
    by_kind<E, 256>(a, paged, splits, st);
}

}  // namespace

void launch_core(const CoreArgs& a, bool paged, int splits, hipStream_t st) {
  if (a.fp16)
    by_dim<f16>(a, paged, splits, st);
  else
    by_dim<bf16>(a, paged, splits, st);
}

}  // namespace cqgdn
