// Attention of many query rows a request over the 4-bit pages: a prompt's rows share the values of a page.
//
// The mathematics, and the rounding of the weights, are those of attn_attend.hip.  Here a workgroup takes 128 rows of one request and key head,
// 32 a wave, and kTokens positions a step.  Its threads convert the step's codes once into K and V tiles of E
// in shared memory, two deep, so that the next step's codes are on their way and being converted while the
// waves multiply.  S^T = K Q^T and O^T = V^T P^T run on 32 x 32 x 16 MFMAs with a row a column, so a lane
// (and its partner 32 lanes on) owns a row: limits, maximum and sum stay in its registers, and S^T's layout
// is already an operand of O^T.
//
// 4096 rows over 8192 positions (16 heads of 128, 4 key heads): 219 us, 941 TFLOP/s; the library's largest products
// reach 1486.  2048 rows over 4096 reach 661, in two parts that the join adds up; with D = 64 636 and 513, whose steps
// hold half of the MFMAs against the same exponentials, masks and barriers; with D = 256, where a SIMD holds one wave
// and its exponentials stand by themselves, 649 and 529.  A step of 32 rows and 64 positions is 32 MFMAs (1024 cycles of the matrix core, each of which keeps the
// SIMD's issue 16 cycles), some 195 VALU instructions, 32 of them exponentials of 8 cycles, and 270 cycles of LDS, which
// eight waves of a CU share: no one of them fills the time, and left out of a copy each takes 7 to 17% with it.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attn_kernels.hpp"
#include "attn_kv4.hpp"
#include "attn_plan.hpp"

namespace cqgdn {
namespace {

constexpr int kRows = 128;  // of a workgroup, 32 a wave
constexpr int kEarly = 4;   // MFMA operands read from LDS ahead of their use: a read's latency is that of four MFMAs

typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// Positions a step, of which 256 threads convert kPiece values of K and of V each.
template <int D>
constexpr int kTokens = D == 256 ? 32 : 64;
template <int D>
constexpr int kPiece = kTokens<D> * D / 256;

// K rows are 16 bytes longer than their values: read 16 bytes a lane, 16 rows at a time, they meet all 64 banks
// once.  V is read by quads of rows and 64 bytes of each; its 16-byte column c lies at v_column(row, c), the
// same for rows 4 apart, so that those meet all banks once as well.  Both are written 16 bytes a lane, every
// fourth column, again without a bank met twice.
template <int D>
constexpr int kStrideK = D + 8;
template <int D>
__device__ __forceinline__ int v_column(int row, int c) {
  if constexpr (D == 64) return c ^ (4 * ((row >> 1) & 1)) ^ ((row >> 1) & 1);
  return c ^ (5 * (row & 3)) ^ (D == 256 ? (c >> 4) << 1 : 0);
}

// a thread's codes of a step's K or V and their scale byte
template <int D>
struct Piece {
  uint32_t w[kPiece<D> / 8];
  uint32_t s;
};
// from a page's buffer: a lane's offsets and the scalar ones of the step's first position
template <int D>
__device__ __forceinline__ Piece<D> fetch(__amdgpu_buffer_rsrc_t page, int code, int code0, int scale, int scale0) {
  Piece<D> x;
  if constexpr (kPiece<D> == 16) {
    const auto w = __builtin_amdgcn_raw_buffer_load_b64(page, code, code0, 0);
    x.w[0] = w[0];
    x.w[1] = w[1];
  } else {
    const u32x4 w = buf_ld16<u32x4>(page, code, code0);
#pragma unroll
    for (int e = 0; e < 4; ++e) x.w[e] = w[e];
  }
  x.s = __builtin_amdgcn_raw_buffer_load_b8(page, scale, scale0, 0);
  return x;
}

template <class E, int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : D == 64 ? 3 : 2) void tile_kernel(AttendArgs a, int tiles, int splits) {
  typedef typename Vec<E>::x8 x8;
  constexpr int TOK = kTokens<D>, VP = kPiece<D>, PV = D / VP, NS = TOK / 32, KQ = D / 16, MT = D / 32;
  constexpr int F = NS * KQ, FV = 2 * NS * MT;  // operands of a step: K's and V's
  constexpr int PARTS = VP / 8, GROUPS = TOK / 16, WAVE_POS = 64 / PV;
  __shared__ __align__(16) E kt[2][TOK * kStrideK<D>];
  __shared__ __align__(16) E vt[2][TOK * D];
  // of the positions each wave converted: whether there is a NaN among the values, and the pieces that have one
  __shared__ __align__(16) int poison[2][4];
  __shared__ uint64_t bad[2][4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n32 = lane & 31, kg = lane >> 5;
  // Launch order: a request's last tiles, which see most, first; every other round of 256 workgroups (one a
  // CU) reversed, so that a CU's workgroups add up to the same
  // The rows of padding behind the requests', "request N", come last: among the others, their workgroups would
  // leave some XCDs with less (prefill of one request 238 us against 229, seven ragged prompts 83 against 75).
  const int each = a.kv_heads * a.N * splits, real_blocks = each * tiles;
  int b = blockIdx.x;
  const bool padding = b >= real_blocks;
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
  const int group = a.group.d, T = (int)a.T;
  const int from = r == 0 ? 0 : min(max(a.starts[r], 0), T);
  const int to = padding ? T : min(max(a.starts[r + 1], from), T);
  const int rows = (to - from) * group, size = 1 << a.page_shift;
  const int room = (int)min((int64_t)a.columns << a.page_shift, (int64_t)kAttendRoom);
  const int token = tid / PV, piece = tid % PV;  // the thread's part of a step
  const uint8_t* const head_base = a.data + (int64_t)h * kv4_page_bytes(size, D);
  const uint64_t stride = (uint64_t)a.kv_heads * kv4_page_bytes(size, D);
  // the exponent's factor, never 0: a masked score stays -infinity; its sign goes with Q
  const float c = fmaxf(fabsf(a.scale) * 1.44269504088896341f, 1.17549435e-38f);
  constexpr float bias = kAttendBias<E>;
  typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
  // the lane's K row of a step, and its piece of V: tokens 4 kg + {0..3, 8..11} at dimension 32 k + n32 come
  // transposed out of quads of lanes
  const int kl = n32 * kStrideK<D> + 8 * kg;
  int vl[MT];
#pragma unroll
  for (int k = 0; k < MT; ++k) {
    const int j = lane & 15, row = 4 * kg + (j >> 2), col = 4 * k + 2 * (lane >> 4 & 1) + (j >> 1 & 1);
    vl[k] = row * D + 8 * v_column<D>(row, col) + 4 * (j & 1);
  }

  for (int tile = tile0; tile * kRows < rows; tile += tiles) {
    const auto limits = [&](int rho, int& lo, int& hi) {
      attend_limits(rho < rows && r < a.N ? a.visible[from + a.group.of(rho)] : 0, a.window, room, lo, hi);
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
    const bool real = rho < rows, active = tile * kRows + 32 * wave < rows;
    int lo, hi;
    limits(rho, lo, hi);
    // the range that all of the wave's rows see, where nothing is masked
    int low = lo, high = real ? hi : INT32_MAX;
#pragma unroll
    for (int i = 1; i < 32; i <<= 1) {
      low = max(low, __shfl_xor(low, i, 64));
      high = min(high, __shfl_xor(high, i, 64));
    }
    low = __builtin_amdgcn_readfirstlane(low);
    high = __builtin_amdgcn_readfirstlane(high);
    const int row_t = real ? a.group.of(rho) : 0, t = from + row_t, head = h * group + (real ? rho - row_t * group : 0);
    x8 qf[KQ];  // lane (n32, kg): row n32, dimensions 16 i + 8 kg ..
    {
      const E* q = static_cast<const E*>(a.q) + t * a.q_token + head * a.q_head + 8 * kg;
#pragma unroll
      for (int i = 0; i < KQ; ++i) {
        u32x4 w = real ? *reinterpret_cast<const u32x4*>(q + 16 * i) : u32x4{0, 0, 0, 0};
        if (a.scale < 0.f) w ^= 0x80008000u;
        qf[i] = __builtin_bit_cast(x8, w);
      }
    }
    f32x16 o[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) o[i] = f32x16{};
    float m = hi > 0 ? -INFINITY : 0.f, l = 0.f;
    uint32_t nan = 0;  // blocks of 32 dimensions in which the row sees a NaN value

    const int begin = last > 0 ? first & ~(TOK - 1) : 0;
    const int steps = (last - begin + TOK - 1) / TOK, per = (steps + splits - 1) / splits;
    const int n = min(steps, (s + 1) * per) - s * per, pos0 = begin + s * per * TOK;

    // the block table's entries for the 16 positions each of step j, one a lane
    const auto entries = [&](int j) {
      const int column = (pos0 + j * TOK + 16 * (lane & (GROUPS - 1))) >> a.page_shift;
      return j < n && column < a.columns ? a.tables[r * a.table_stride + column] : -1;
    };
    Piece<D> kn, vn;
    const int code = lane / PV * (D / 2) + VP / 2 * piece, scale = lane / PV * (D / 32) + piece * VP / 32;
    // step j's codes of the wave's positions, which one page holds; one that is hidden reads as zeros.  Returns
    // which of the step's 16 positions are shown.
    const auto fetch_step = [&](int table, int j) {
      const uint32_t page = __builtin_amdgcn_readlane(table, wave * WAVE_POS / 16);
      const bool ok = page < a.page_count;
      const __amdgpu_buffer_rsrc_t rs = buf_rsrc(head_base + (ok ? page * stride : 0), ok ? kv4_page_bytes(size, D) : 0);
      const int at = (pos0 + j * TOK + wave * WAVE_POS) & (size - 1);
      const auto place = [&](int offset) { return ok ? offset : 0; };  // scalar: buf_rsrc's rule
      kn = fetch<D>(rs, code, place(at * (D / 2)), scale, place(size * D + at * (D / 32)));
      vn = fetch<D>(rs, code, place((size + at) * (D / 2)), scale, place(size * D + (size + at) * (D / 32)));
      return (int)__ballot((uint32_t)table < a.page_count) & ((1 << GROUPS) - 1);
    };
    // those codes become step j's K and V tiles, PARTS parts of each.  Where the step reaches beyond what the
    // rows see, a position that no row sees is zero, and so is a NaN value: it goes to the rows that see it by `nan`.
    float kscale, vscale;
    E* const kw = kt[0] + token * kStrideK<D> + VP * piece;
    int vw[PARTS];
#pragma unroll
    for (int e = 0; e < PARTS; ++e) vw[e] = token * D + 8 * v_column<D>(token, PARTS * piece + e);
    const auto begin_convert = [&](int j) {
      uint64_t nans = __ballot(vn.s == 255);
      const int pos = pos0 + j * TOK;
      if (nans != 0 || pos < first || pos + TOK > last) {
        const bool any = pos + token >= first && pos + token < last;
        nans = __ballot(any && vn.s == 255);
        if (!any || vn.s == 255) {
          vn.s = 0;
#pragma unroll
          for (int e = 0; e < PARTS; ++e) vn.w[e] = 0;
        }
        if (lane == 0) bad[j & 1][wave] = nans;
      }
      if (lane == 0) poison[j & 1][wave] = nans != 0;
      kscale = kv4_scale(kn.s);
      vscale = kv4_scale(vn.s);
    };
    const auto convert = [&](int j, int e) {
      if (e < PARTS)
        st8(kw + (j & 1) * (TOK * kStrideK<D>) + 8 * e, kv4_values<E>(kn.w[e], kscale));
      else
        st8(vt[j & 1] + vw[e - PARTS], kv4_values<E>(vn.w[e - PARTS], vscale));
    };
    f32x16 sc[NS];
    // the weights of 32 positions, two a part, in the order of their scores
    uint32_t pw[NS][8];
    float base, sum;
    const auto begin_weights = [&]() {
      base = bias - (m == -INFINITY ? 0.f : m);
      sum = 0.f;
    };
    const auto weights = [&](int u, int i) {
      typedef float f32x2 __attribute__((ext_vector_type(2)));
      typedef E x2 __attribute__((ext_vector_type(2)));
      f32x2 p;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[u][2 * i + e], c, base));
        sum += p[e];
      }
      pw[u][i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(p, x2));
    };
    // hidden positions leave the scores
    const auto mask = [&](int u, int pos, int shown) {
      if (shown == (1 << GROUPS) - 1 && pos >= low && pos + TOK <= high) return;
      const int lo0 = lo - pos - 4 * kg, hi0 = hi - pos - 4 * kg;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int at = 32 * u + 8 * (e >> 2) + (e & 3);
        if ((int)(at < lo0) | (int)(at >= hi0) | (int)!(shown >> (2 * u + (e >> 3)) & 1)) sc[u][e] = -INFINITY;
      }
    };
    // where the weights have grown too large, or are a row's first, its maximum moves and they are made again
    const auto settle = [&](int u) {
      bool large = sum > kAttendLimit<E> || m == -INFINITY;
      if (__any(large)) {
        large = __shfl_xor((int)large, 32, 64) || large;  // the two lanes of a row
        float top = sc[u][0];
#pragma unroll
        for (int e = 1; e < 16; ++e) top = fmaxf(top, sc[u][e]);
        top = fmaxf(top, __shfl_xor(top, 32, 64)) * c;
        if (large && top > m) {
          const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
          m = top;
          l *= f;
#pragma unroll
          for (int k = 0; k < MT; ++k) o[k] *= f;
        }
        begin_weights();
#pragma unroll
        for (int i = 0; i < 8; ++i) weights(u, i);
      }
      l += sum;
    };

    if (n > 0) {
      int shown = fetch_step(entries(0), 0), shown1 = 0;
      begin_convert(0);
#pragma unroll
      for (int e = 0; e < 2 * PARTS; ++e) convert(0, e);
      shown1 = fetch_step(entries(1), 1);
      int table = entries(2);
      __syncthreads();
#pragma unroll 1
      for (int j = 0; j < n; ++j) {
        if (active) {
          const E* const kp = kt[j & 1] + kl;
          const E* const vp = vt[j & 1];
          x8 kf[F], vf[FV];
          const auto value = [&](int i) {  // positions 16 (i / MT), dimensions 32 (i % MT)
            const E* p = vp + vl[i % MT] + i / MT * 16 * D;
            const i16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)p);
            const i16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(p + 8 * D));
            vf[i] = __builtin_bit_cast(x8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
          };
#pragma unroll
          for (int i = 0; i < 2 * kEarly; ++i) kf[i] = ld8(kp + i / KQ * 32 * kStrideK<D> + i % KQ * 16);
          const int4 poisoned = *reinterpret_cast<const int4*>(poison[j & 1]);
          const int pos = pos0 + j * TOK;
          constexpr int H = FV / NS;  // operands of V for 32 positions
          const auto score = [&](int u, int i) {
            if (i == 0) sc[u] = f32x16{};
            sc[u] = mfma32(kf[u * KQ + i], qf[i], sc[u]);
            const int k = u * KQ + i + 2 * kEarly;
            if (k < F) kf[k] = ld8(kp + k / KQ * 32 * kStrideK<D> + k % KQ * 16);
          };
          const auto gather = [&](int u, int i) {
            const int w = i / MT * 4;
            const x8 p = __builtin_bit_cast(x8, u32x4{pw[u][w], pw[u][w + 1], pw[u][w + 2], pw[u][w + 3]});
            o[i % MT] = mfma32(vf[u * H + i], p, o[i % MT]);
          };
          // An MFMA leaves the wave's issue free for about as long as two weights take.  So the first 32
          // positions' weights stand between the second's scores, the second's between the first's products
          // with V, and the next step's conversions between the last.
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int i = 0; i < KQ; ++i) {
            score(0, i);
            __builtin_amdgcn_sched_barrier(0);
          }
          mask(0, pos, shown);
          begin_weights();
          if constexpr (NS == 2) {
#pragma unroll
            for (int i = 0; i < KQ; ++i) {
              score(1, i);
#pragma unroll
              for (int e = i * 8 / KQ; e < (i + 1) * 8 / KQ; ++e) weights(0, e);
#pragma unroll
              for (int e = i * H / KQ; e < (i + 1) * H / KQ; ++e) value(e);
              __builtin_amdgcn_sched_barrier(0);
            }
            settle(0);
            mask(1, pos, shown);
            begin_weights();
#pragma unroll
            for (int i = 0; i < H; ++i) {
              gather(0, i);
#pragma unroll
              for (int e = i * 8 / H; e < (i + 1) * 8 / H; ++e) weights(1, e);
              value(H + i);
              __builtin_amdgcn_sched_barrier(0);
            }
          } else {
#pragma unroll
            for (int i = 0; i < kEarly; ++i) value(i);
#pragma unroll
            for (int e = 0; e < 8; ++e) weights(0, e);
          }
          settle(NS - 1);
          begin_convert(j + 1);  // beyond the last step: of codes that nothing reads
#pragma unroll
          for (int i = 0; i < H; ++i) {
            gather(NS - 1, i);
            if (NS == 1 && i + kEarly < H) value(i + kEarly);
#pragma unroll
            for (int e = i * 2 * PARTS / H; e < (i + 1) * 2 * PARTS / H; ++e) convert(j + 1, e);
            __builtin_amdgcn_sched_barrier(0);
          }
          if (__builtin_amdgcn_readfirstlane(poisoned.x | poisoned.y | poisoned.z | poisoned.w)) {
#pragma unroll 1
            for (int w = 0; w < 4; ++w)
#pragma unroll 1
              for (uint64_t y = poison[j & 1][w] ? bad[j & 1][w] : 0; y; y &= y - 1) {
                const int i = 64 * w + __builtin_ctzll(y), at = pos0 + j * TOK + i / PV;
                nan |= at >= lo && at < hi ? 1u << (i % PV * VP / 32) : 0u;
              }
          }
        } else {
          begin_convert(j + 1);
#pragma unroll
          for (int e = 0; e < 2 * PARTS; ++e) convert(j + 1, e);
        }
        shown = shown1;
        shown1 = fetch_step(table, j + 2);
        table = entries(j + 3);
        __syncthreads();
      }
    }
    l += __shfl_xor(l, 32, 64);
    if (__any(nan != 0)) {
#pragma unroll
      for (int k = 0; k < MT; ++k)
        if (nan >> k & 1) o[k] = f32x16{} + __builtin_nanf("");
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
    __syncthreads();
  }
}

template <class E, int D>
void launch_dim(const AttendArgs& a, int splits, hipStream_t st) {
  const int64_t each = std::max<int64_t>(1, (int64_t)a.N * a.kv_heads * splits);
  const int64_t wanted = ((int64_t)a.max_queries * (a.heads / a.kv_heads) + kRows - 1) / kRows;
  const int tiles = (int)std::max<int64_t>(1, std::min<int64_t>(wanted, (1 << 23) / each));
  const int64_t blocks = (int64_t)a.N * a.kv_heads * splits * tiles + (int64_t)a.kv_heads * std::min(tiles, 16);
  tile_kernel<E, D><<<(unsigned)blocks, 256, 0, st>>>(a, tiles, splits);
}

template <class E>
void by_dim(const AttendArgs& a, int splits, hipStream_t st) {
  if (a.D == 64)
    launch_dim<E, 64>(a, splits, st);
  else if (a.D == 128)
    launch_dim<E, 128>(a, splits, st);
  else
    launch_dim<E, 256>(a, splits, st);
}

}  // namespace

void launch_attend_tiles(const AttendArgs& a, int splits, hipStream_t st) {
  if (a.fp16)
    by_dim<f16>(a, splits, st);
  else
    by_dim<bf16>(a, splits, st);
}

}  // namespace cqgdn
