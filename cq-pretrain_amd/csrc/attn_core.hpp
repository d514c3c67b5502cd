// What the attention kernels over 16-bit rows share: tiles of rows in LDS, their MFMA operands, the scores' cap and
// bias, and values that are not finite.
//
// S^T = K Q^T, O^T = V^T P^T and the products of the gradients run on 32 x 32 x 16 MFMAs, lane (n32, kg) of
// 32 columns and two halves:
//   A (32 x 16): row n32, k = 8 kg .. 8 kg + 7;  B (16 x 32): column n32, the same k;
//   C (32 x 32): column n32, element e is row 8 (e >> 2) + 4 kg + (e & 3)
// so that elements 8 b .. 8 b + 7 of a C are the B operand of a product over its rows 16 b .. 16 b + 15, whose k runs
// 4 kg + {0 .. 3, 8 .. 11}: the A operand is read from a tile in that order, transposed.
#pragma once
#include "attn_kernels.hpp"
#include "attn_kv4.hpp"
#include "gdn_common.hpp"

namespace cqgdn {

typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
// A tile of 64 rows [D] in LDS, as asynchronous loads write it: 1024 bytes an instruction, side by side, the lanes anywhere
// in memory.  Such a block holds 4 chunks (of 16 bytes) of 16 rows, a row's side by side and in their order: the memory
// pipeline then takes a row's 64 bytes as one request (chunks put in another order are a request each, and cost the
// forward pass of 9216 rows 447 us against 412).  Each 16 rows' blocks lie 16 bytes further than the last's.  The rows that an MFMA
// takes as its 32 come from all four: row m of the u-th 32 is tile row 16 (m >> 2 & 3) + 8 u + 4 (m >> 4) + (m & 3).
// 16 rows read at the same chunk, and 4 rows at 4 neighbouring chunks (the transposed reads), meet all 64 banks once, and
// but for two offsets of the lane every place in the tile is a constant.
constexpr int kTile = 64;  // rows
template <int D>
constexpr int kTileRows16 = 16 * D + 8;  // elements from 16 rows to the next
template <int D>
constexpr int kTileSize = 4 * kTileRows16<D>;
template <int D>
__host__ __device__ constexpr int tile_at(int row, int chunk) {  // in elements
  return row / 16 * kTileRows16<D> + chunk / 4 * 512 + (row & 15) * 32 + (chunk & 3) * 8;
}
// the tile row of element e of the u-th C, without the lane's 16 kg
__host__ __device__ constexpr int c_row(int u, int e) { return 32 * (e >> 2 & 1) + 8 * u + 4 * (e >> 3) + (e & 3); }

template <class E, int D>
struct TileOperands {
  typedef typename Vec<E>::x8 x8;
  int row, col;  // of the lane, in elements
  __device__ __forceinline__ TileOperands(int lane) {
    const int m = lane & 31, kg = lane >> 5, j = lane & 15;
    row = tile_at<D>(16 * (m >> 2 & 3) + 4 * (m >> 4) + (m & 3), kg);
    col = tile_at<D>(16 * kg + (j >> 2), 2 * (lane >> 4 & 1) + (j >> 1 & 1)) + 4 * (j & 1);
  }
  // the u-th 32 rows, dimensions 16 i + 8 kg ..
  __device__ __forceinline__ x8 rows(const E* tile, int u, int i) const { return ld8(tile + row + tile_at<D>(8 * u, 2 * i)); }
  // dimension 32 m + n32 of the rows of elements 8 b .. 8 b + 7 of the u-th C
  __device__ __forceinline__ x8 columns(const E* tile, int u, int b, int m) const {
    typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
    const E* p = tile + col + tile_at<D>(8 * u + 4 * b, 4 * m);
    const i16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)p);
    const i16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(p + 2 * kTileRows16<D>));
    return __builtin_bit_cast(x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
  }
};

// N blocks of a tile on their way: lane l's 16 bytes of `from` + `off` + 64 i (bytes) land at `lds` + 1024 i + 16 l.  In
// assembly because the compiler, which does not tell the tiles of a pair from each other, puts a wait for all that is on
// its way before every read of the other one (the forward pass of 9216 rows spent 61% of its time in that wait); tiles_ready()
// is the wait that is needed.  Nothing is returned in registers.  An instruction's offset moves both addresses.
template <int N>
__device__ __forceinline__ void load_blocks(const void* from, uint32_t off, void* lds) {
  // the same for all lanes, in scalar registers
  const uint32_t at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_void_ptr)lds);
  const uintptr_t x = reinterpret_cast<uintptr_t>(from);
  const uintptr_t base = (uintptr_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(x >> 32)) << 32 |
                         (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)x);
#define CQGDN_LOAD(m0, more) "s_mov_b32 m0, " m0 "\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" more "\n\t"
  static_assert(N == 1 || N == 2 || N == 4 || N == 8, "blocks a wave");
  if constexpr (N == 1) {
    asm volatile(CQGDN_LOAD("%2", "") ::"v"(off), "s"(base), "s"(at) : "memory", "m0");
  } else if constexpr (N == 2) {
    asm volatile(CQGDN_LOAD("%2", "") CQGDN_LOAD("%3", " offset:64") ::"v"(off), "s"(base), "s"(at), "s"(at + 960)
                 : "memory", "m0");
  } else {
    asm volatile(CQGDN_LOAD("%2", "") CQGDN_LOAD("%3", " offset:64") CQGDN_LOAD("%4", " offset:128")
                     CQGDN_LOAD("%5", " offset:192") ::"v"(off),
                 "s"(base), "s"(at), "s"(at + 960), "s"(at + 1920), "s"(at + 2880)
                 : "memory", "m0");
    if constexpr (N == 8) load_blocks<4>(static_cast<const char*>(from) + 256, off, static_cast<char*>(lds) + 4096);
  }
#undef CQGDN_LOAD
}
// 16 rows of a tile, by one wave: row lane / 4 of `rows` (the wave's, from dimension 0 on), `offset` elements from there
template <class E, int D>
__device__ __forceinline__ void load_rows16(const E* rows, uint32_t offset, E* tile, int wave, int lane) {
  load_blocks<D / 32>(rows, (offset + 8 * (lane & 3)) * sizeof(E), tile + wave * kTileRows16<D>);
}
// What the workgroup's waves have asked for has arrived, and all have read what they wanted.
__device__ __forceinline__ void tiles_ready() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// ---- values that are not finite -----------------------------------------------------------------------
// 0 x infinity and 0 x NaN are NaN, so a value that a row does not see must not meet its weight 0 in an MFMA.  Looking
// for such values in every step whose rows do not all see all of it would cost as much as the step.  Instead a workgroup
// looks at its sums when it is done: if one is not finite it goes through its steps once more, carefully: there, values
// that are not finite go in as 0 and are added afterwards, lane by lane, to those that see them.
template <int N>
__device__ __forceinline__ bool any_not_finite(const f32x16 (&x)[N]) {
  float zero[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) zero[e & 3] = __builtin_fmaf(x[i][e], 0.f, zero[e & 3]);
  return !((zero[0] + zero[1]) + (zero[2] + zero[3]) == 0.f);
}
template <class E>
__device__ __forceinline__ uint32_t odd_values(u32x4 w) {
  constexpr uint32_t exponent = std::is_same<E, f16>::value ? 0x7C007C00u : 0x7F807F80u;
  constexpr uint32_t one = std::is_same<E, f16>::value ? 0x04000400u : 0x00800080u;
  uint32_t any = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) any |= (w[e] & exponent) + one;
  return any & 0x80008000u;
}
template <class E, class X8>
__device__ __forceinline__ X8 finite_values(X8 x) {
  u32x4 w = __builtin_bit_cast(u32x4, x);
  constexpr uint32_t exponent = std::is_same<E, f16>::value ? 0x7C007C00u : 0x7F807F80u;
  constexpr uint32_t one = std::is_same<E, f16>::value ? 0x04000400u : 0x00800080u;
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] &= ~(((((w[e] & exponent) + one) & 0x80008000u) >> 15) * 0xFFFFu);
  return __builtin_bit_cast(X8, w);
}
// whether the tile holds one
template <class E, int D>
__device__ __forceinline__ bool tile_is_odd(const E* tile, int lane) {
  uint32_t any = 0;
#pragma unroll
  for (int b = 0; b < 4; ++b)
#pragma unroll
    for (int i = 0; i < D / 32; ++i) any |= odd_values<E>(*reinterpret_cast<const u32x4*>(tile + b * kTileRows16<D> + 512 * i + 8 * lane));
  return __any(any != 0);
}
// acc (dimension 32 (m0 + m) + 8 (e >> 2) + 4 kg + (e & 3) of the lane's column) += what the tile's rows hold beyond finite
// values, of the rows that sees(row) allows the lane
template <class E, int D, int MT, class Sees>
__device__ __forceinline__ void add_odd(const E* tile, f32x16 (&acc)[MT], int lane, Sees sees, int m0 = 0) {
  const int kg = lane >> 5;
#pragma unroll 1
  for (int i = 0; i < kTile; ++i) {
    const bool seen = sees(i);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) {
        const int d = 32 * (m0 + m) + 8 * e4 + 4 * kg;
        const auto x = ld4(tile + tile_at<D>(i, d >> 3) + (d & 7));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float f = (float)x[e];
          if (seen && !(f - f == 0.f)) acc[m][4 * e4 + e] += f;
        }
      }
  }
}

// A row whose scores are all -infinity is NaN, as 0 / 0 is.  A part of it alone may be such a part of a row that is not:
// it leaves the maximum -infinity and this as its sum, which the join multiplies with exp2(-infinity - the row's maximum):
// 0 beside parts with finite scores, NaN where there is none.
constexpr float kNoWeight = -1.f;
// whether a page holds any of the positions [from, to) of request r
__device__ __forceinline__ bool pages_hold(const CoreArgs& a, int r, int from, int to) {
  for (int column = from >> a.page_shift; from < to && column <= (to - 1) >> a.page_shift; ++column)
    if ((uint32_t)a.tables[r * a.table_stride + column] < a.page_count) return true;
  return false;
}

// ---- scores -------------------------------------------------------------------------------------------
// A score x = scale q.k becomes u = cap tanh(x / cap) - slope |distance|, in units of log2 e throughout.  With
// r = 1 / (1 + e^(2 x / cap)) the tanh is 1 - 2 r (an exponential and a reciprocal; off by 2^-23 of the cap), and its
// derivative 4 (r - r^2).
struct Bend {
  float c, cap, slope;  // scale or 2 scale / cap, cap, slope, each times log2 e; cap 0: none
  __device__ __forceinline__ Bend(float scale, float cap_, const float* slopes, int head) {
    constexpr float log2e = 1.44269504088896341f;
    c = cap_ > 0.f ? 2.f * scale / cap_ * log2e : scale * log2e;
    cap = cap_ * log2e;
    slope = slopes ? slopes[head] * log2e : 0.f;
  }
  // -r, which grows with x
  __device__ __forceinline__ float less_r(float x) const {
    return __builtin_amdgcn_rcpf(-1.f - __builtin_amdgcn_exp2f(x * c));
  }
  // the capped score plus what is added to it less the cap, and a quarter of its derivative by the uncapped one
  __device__ __forceinline__ float capped(float x, float more) const { return __builtin_fmaf(2.f * cap, less_r(x), more); }
  __device__ __forceinline__ float capped(float x, float more, float& rate) const {
    const float r = less_r(x);
    rate = __builtin_fmaf(r, -r, -r);
    return __builtin_fmaf(2.f * cap, r, more);
  }
};

// Distances of packed rows are counted in fp32: keys lie below 2^24, and a position beyond it counts as that, so that
// every kernel has the same distance, not rounded.
constexpr int kFarthest = 1 << 24;
__device__ __forceinline__ int within_reach(int position) { return min(max(position, -kFarthest), kFarthest); }

// f with whether scores are capped and whether they are biased, as types
template <class F>
void by_scores(const CoreArgs& a, F f) {
  if (a.cap > 0.f)
    a.slopes ? f(std::true_type{}, std::true_type{}) : f(std::true_type{}, std::false_type{});
  else
    a.slopes ? f(std::false_type{}, std::true_type{}) : f(std::false_type{}, std::false_type{});
}

// What the keys' gradients need of 64 rows of a key head, as the queries' gradients leave it.
struct RowBlock {
  float lse[64], delta[64];     // cap less log2 sum of exp2, and the gradient of lse less sum p dy.v: what is added
  int lo[64], hi[64];           // the keys that the row sees
  float stands[64], slope[64];  // with a bias: the row's position, its head's slope times log2 e
};
// The keys that any of 64 rows sees, [first, last) (first = INT32_MAX, last = 0 where none sees any), and those that
// all of them see, [low, high).
struct RowRange {
  int first, last, low, high;
};

}  // namespace cqgdn
