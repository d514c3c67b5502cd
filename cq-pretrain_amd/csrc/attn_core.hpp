// What the attention kernels over 16-bit rows share: tiles of rows in LDS, their MFMA operands, the scores' cap and
// bias, and values that are not finite.
//
// S^T = K Q^T, O^T = V^T P^T and the products of the gradients run on 32 x 32 x 16 MFMAs, lane (n32, kg) of
// 32 columns and two halves:
//   A (32 x 16): row n32, k = 8 kg .. 8 kg + 7;  B (16 x 32): column n32, the same k;
//   C (32 x 32): column n32, element e is row 8 (e >> 2) + 4 kg + (e & 3)
// so that elements 8 i .. 8 i + 7 of a C are the B operand of a product over rows 16 i .. 16 i + 15, whose k runs
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
// the row of a C's element, without the lane's 4 kg
__host__ __device__ constexpr int c_row(int e) { return 8 * (e >> 2) + (e & 3); }

// A tile of rows [n][D] in LDS, as global loads write it: 1024 bytes an instruction, side by side, so there is no
// room between rows.  The 16-byte chunk c of a row lies at c ^ turn(row): 16 rows read at the same chunk, and 4 rows
// at 4 neighbouring chunks (the transposed reads), then meet all 64 banks once.
template <int D>
__device__ __forceinline__ int tile_turn(int row) {
  return D == 64 ? (row >> 1 & 1) << 2 | (row >> 2 & 3) : (row & 3) << 2 | (row >> 2 & 3);
}
template <class E, int D>
struct TileOperands {
  typedef typename Vec<E>::x8 x8;
  int row[D / 16], col[2][D / 32];  // of the lane, in elements
  __device__ __forceinline__ TileOperands(int lane) {
    const int n32 = lane & 31, kg = lane >> 5, j = lane & 15;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) row[i] = n32 * D + 8 * ((2 * i) ^ kg ^ tile_turn<D>(n32));
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int m = 0; m < D / 32; ++m) {
        const int r = 4 * kg + 8 * s + (j >> 2);
        col[s][m] = r * D + 8 * ((4 * m + 2 * (lane >> 4 & 1) + (j >> 1 & 1)) ^ tile_turn<D>(r)) + 4 * (j & 1);
      }
  }
  // rows 32 u + n32, dimensions 16 i + 8 kg ..
  __device__ __forceinline__ x8 rows(const E* tile, int u, int i) const { return ld8(tile + 32 * u * D + row[i]); }
  // dimension 32 m + n32 of the rows 16 b + 4 kg + {0 .. 3, 8 .. 11}
  __device__ __forceinline__ x8 columns(const E* tile, int b, int m) const {
    typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
    const i16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(tile + 16 * b * D + col[0][m]));
    const i16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(tile + 16 * b * D + col[1][m]));
    return __builtin_bit_cast(x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
  }
};
// rows that one instruction of a wave loads, and the lane's row and chunk of those from row0 (a multiple of kLoadRows)
template <int D>
constexpr int kLoadRows = 512 / D;
template <int D>
__device__ __forceinline__ int load_row(int lane) { return lane / (D / 8); }
template <int D>
__device__ __forceinline__ int load_chunk(int lane, int row) { return (lane % (D / 8)) ^ tile_turn<D>(row); }

// ---- values that are not finite -----------------------------------------------------------------------
// 0 x infinity and 0 x NaN are NaN, so a value that a row does not see must not meet its weight 0 in an MFMA.  Where a
// step's rows do not all see all of it, its operands are looked through; if one holds such a value, it goes in as 0
// and is added afterwards, lane by lane, to those that see it.
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
// whether the tile's first 16 B rows hold one
template <class E, int D, int B>
__device__ __forceinline__ bool tile_is_odd(const E* tile, int lane) {
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < B * 16 * D / 512; ++i) any |= odd_values<E>(*reinterpret_cast<const u32x4*>(tile + 512 * i + 8 * lane));
  return __any(any != 0);
}
// acc (dimension 32 (m0 + m) + c_row(e) + 4 kg of the lane's column) += what the tile's first 16 B rows hold beyond finite
// values, of the rows that sees(row) allows the lane
template <class E, int D, int B, int MT, class Sees>
__device__ __forceinline__ void add_odd(const E* tile, f32x16 (&acc)[MT], int lane, Sees sees, int m0 = 0) {
  const int kg = lane >> 5;
#pragma unroll 1
  for (int i = 0; i < 16 * B; ++i) {
    const bool seen = sees(i);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) {
        const int d = 32 * (m0 + m) + 8 * e4 + 4 * kg;
        const auto x = ld4(tile + i * D + 8 * ((d >> 3) ^ tile_turn<D>(i)) + (d & 7));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float f = (float)x[e];
          if (seen && !(f - f == 0.f)) acc[m][4 * e4 + e] += f;
        }
      }
  }
}

// ---- scores -------------------------------------------------------------------------------------------
// A score x = scale q.k becomes u = cap tanh(x / cap) - slope |distance|, in units of log2 e throughout.  With
// r = 1 / (1 + e^(2 x / cap)) the tanh is 1 - 2 r (an exponential and a reciprocal; off by 2^-23 of the cap), and its
// derivative 4 r (1 - r).
struct Bend {
  float c, cap, slope;  // scale or 2 scale / cap, cap, slope, each times log2 e; cap 0: none
  __device__ __forceinline__ Bend(float scale, float cap_, const float* slopes, int head) {
    constexpr float log2e = 1.44269504088896341f;
    c = cap_ > 0.f ? 2.f * scale / cap_ * log2e : scale * log2e;
    cap = cap_ * log2e;
    slope = slopes ? slopes[head] * log2e : 0.f;
  }
  __device__ __forceinline__ float capped(float x) const {
    return __builtin_fmaf(-2.f * cap, __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * c)), cap);
  }
  // the capped score, and the derivative of it by the uncapped one
  __device__ __forceinline__ float capped(float x, float& rate) const {
    const float r = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * c));
    rate = 4.f * r * (1.f - r);
    return __builtin_fmaf(-2.f * cap, r, cap);
  }
};

// What the keys' gradients need of 32 rows of a key head, as the queries' gradients leave it.
struct RowBlock {
  float lse[32], delta[32];     // log2 sum of exp2, and dy.out less the gradient of lse
  int lo[32], hi[32];           // the keys that the row sees
  float stands[32], slope[32];  // with a bias: the row's position, its head's slope times log2 e
};
// The keys that any of 32 rows sees, [first, last) (first = INT32_MAX, last = 0 where none sees any), and those that
// all of them see, [low, high).
struct RowRange {
  int first, last, low, high;
};

}  // namespace cqgdn
