// Rows of keys and values rounded into the 4-bit pages, and read back.
//
// Of 32 neighbouring values the largest magnitude m sets the scale 2^s: s = floor(log2 m) - 2, so that
// m / 2^s lies in [4, 8), and one more where it lies above 7 (the largest code stands for 6: above 7 the
// cut costs the largest value more than the coarser steps cost the others; over normal values the
// threshold 7 leaves 11.2% rms error, 6 leaves 11.6%, 8 leaves 11.5%).  s stays above -126, so that no
// value read back is subnormal, and at most 125 (13 for fp16 rows), so that none reads back as infinity.  Codes are rounded to nearest even by the conversion instruction.  A
// block with an infinity or NaN is stored as scale byte 255 and reads back as NaN.
#include <hip/hip_runtime.h>

#include "attn_kernels.hpp"
#include "attn_kv4.hpp"

namespace cqgdn {
namespace {

constexpr int kThreads = 256;

template <class E>
constexpr int kTop = 127 + (std::is_same<E, f16>::value ? 13 : 125);  // the largest scale byte

// where a row of the cache lies: page base, and the token's place in the page
struct Place {
  uint8_t* page;
  int at;
};
__device__ __forceinline__ Place place(const RowsArgs& a, int slot, int h) {
  const int size = 1 << a.page_shift;
  return {a.data + ((int64_t)(slot >> a.page_shift) * a.heads + h) * kv4_page_bytes(size, a.D), slot & (size - 1)};
}

// Rows go through the launch by 16 tokens of a head, whose codes lie side by side where a prompt fills its pages
// (one token's heads lie a page apart: 8191 tokens of 16 heads written and read 44.5 us by those, 42.9 by these).
__device__ __forceinline__ bool token_head(const RowsArgs& a, uint32_t row, int& t, int& h) {
  const int sixteen = (int)(row >> 4), group = a.by_heads.of(sixteen);
  t = group * 16 + (int)(row & 15);
  h = sixteen - group * a.heads;
  return t < a.T;
}

// A thread rounds 8 values (16 bytes in, 4 out), four neighbours share a block's maximum.
template <class E>
__global__ __launch_bounds__(kThreads) void write_kernel(RowsArgs a, int row_threads_shift) {
  const int w = blockIdx.y, lane = threadIdx.x & ((1 << row_threads_shift) - 1);
  int t, h;
  if (!token_head(a, (blockIdx.x * (uint32_t)kThreads + threadIdx.x) >> row_threads_shift, t, h))
    return;  // whole rows leave: the four lanes of a block stay together
  typedef typename Vec<E>::x8 x8;
  const E* src = static_cast<const E*>(w ? a.v : a.k) + t * a.token[w] + h * a.head[w] + 8 * lane;
  const f32x8 x = cvtf8(*reinterpret_cast<const x8*>(src));  // on its way beside the slot
  const int slot = a.slots[t];
  if (slot < 0 || slot >= a.slot_count) return;
  uint32_t top = 0;  // magnitudes order as their bits do, infinities and NaN above the rest
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float f = x[j];  // a copy: __builtin_bit_cast of a vector's element takes the first one
    top = max(top, __builtin_bit_cast(uint32_t, f) & 0x7FFFFFFFu);
  }
  top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0xB1, 0xF, 0xF, true));  // lane ^ 1
  top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0x4E, 0xF, 0xF, true));  // lane ^ 2
  const bool finite = top < 0x7F800000u;
  const int byte = finite ? min(max((int)(top >> 23) - 2 + ((top & 0x7FFFFFu) > 0x600000u), 2), kTop<E>) : 255;
  const float scale = __builtin_bit_cast(float, (uint32_t)byte << 23);
  uint32_t code = 0;
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[0], x[1], scale, 0);
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[2], x[3], scale, 1);
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[4], x[5], scale, 2);
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[6], x[7], scale, 3);
  if (!finite) code = 0;
  const Place p = place(a, slot, h);
  const int size = 1 << a.page_shift;
  uint8_t* codes = p.page + (w ? size * (a.D / 2) : 0) + p.at * (a.D / 2);
  uint8_t* scales = p.page + size * a.D + (w ? size * (a.D / 32) : 0) + p.at * (a.D / 32);
  reinterpret_cast<uint32_t*>(codes)[lane] = code;
  if ((lane & 3) == 0) scales[lane >> 2] = (uint8_t)byte;
}

template <class E>
__global__ __launch_bounds__(kThreads) void read_kernel(RowsArgs a, int row_threads_shift) {
  const int w = blockIdx.y, lane = threadIdx.x & ((1 << row_threads_shift) - 1);
  int t, h;
  if (!token_head(a, (blockIdx.x * (uint32_t)kThreads + threadIdx.x) >> row_threads_shift, t, h)) return;
  const int slot = a.slots[t];
  typename Vec<E>::x8 y = zero8v<E>();
  if (slot >= 0 && slot < a.slot_count) {
    const Place p = place(a, slot, h);
    const int size = 1 << a.page_shift;
    const uint8_t* codes = p.page + (w ? size * (a.D / 2) : 0) + p.at * (a.D / 2);
    const uint8_t* scales = p.page + size * a.D + (w ? size * (a.D / 32) : 0) + p.at * (a.D / 32);
    y = kv4_values<E>(reinterpret_cast<const uint32_t*>(codes)[lane], kv4_scale(scales[lane >> 2]));
  }
  st8(static_cast<E*>(w ? a.v_out : a.k_out) + ((int64_t)t * a.heads + h) * a.D + 8 * lane, y);
}

}  // namespace

void launch_kv4_write(const RowsArgs& a, hipStream_t st) {
  const int shift = __builtin_ctz(a.D / 8);
  const dim3 grid((unsigned)((((int64_t)(a.T + 15) / 16 * 16 * a.heads << shift) + kThreads - 1) / kThreads), 2);
  if (a.fp16)
    write_kernel<f16><<<grid, kThreads, 0, st>>>(a, shift);
  else
    write_kernel<bf16><<<grid, kThreads, 0, st>>>(a, shift);
}

void launch_kv4_read(const RowsArgs& a, hipStream_t st) {
  const int shift = __builtin_ctz(a.D / 8);
  const dim3 grid((unsigned)((((int64_t)(a.T + 15) / 16 * 16 * a.heads << shift) + kThreads - 1) / kThreads), 2);
  if (a.fp16)
    read_kernel<f16><<<grid, kThreads, 0, st>>>(a, shift);
  else
    read_kernel<bf16><<<grid, kThreads, 0, st>>>(a, shift);
}

}  // namespace cqgdn
