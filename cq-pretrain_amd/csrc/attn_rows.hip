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
// (one token's heads lie a page apart: 8191 tokens of 16 heads written
// and read 44.5 us by those, 42.9 by these, 41.0 with four rows a thread: 4.1 TB/s).
__device__ __forceinline__ bool token_head(const RowsArgs& a, uint32_t row, int& t, int& h) {
  const int sixteen = (int)(row >> 4), group = a.by_heads.of(sixteen);
  t = group * 16 + (int)(row & 15);
  h = sixteen - group * a.heads;
  return t < a.T;
}

// A thread rounds 8 values (16 bytes in, 4 out), four neighbours share a block's maximum; it takes N rows of them,
// whose loads are all under way at once.
template <class E, int N>
__global__ __launch_bounds__(kThreads) void write_kernel(RowsArgs a, int row_threads_shift) {
  typedef typename Vec<E>::x8 x8;
  const int w = blockIdx.y, lane = threadIdx.x & ((1 << row_threads_shift) - 1), size = 1 << a.page_shift;
  int h[N], slot[N];
  x8 raw[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    int t;
    slot[i] = -1;
    raw[i] = zero8v<E>();
    if (token_head(a, ((blockIdx.x * N + i) * (uint32_t)kThreads + threadIdx.x) >> row_threads_shift, t, h[i])) {
      slot[i] = a.slots[t];
      raw[i] = *reinterpret_cast<const x8*>(static_cast<const E*>(w ? a.v : a.k) + t * a.token[w] + h[i] * a.head[w] + 8 * lane);
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (slot[i] < 0 || slot[i] >= a.slot_count) continue;  // whole rows: the four lanes of a block stay together
    const f32x8 x = cvtf8(raw[i]);
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
    const Place p = place(a, slot[i], h[i]);
    uint8_t* codes = p.page + (w ? size * (a.D / 2) : 0) + p.at * (a.D / 2);
    uint8_t* scales = p.page + size * a.D + (w ? size * (a.D / 32) : 0) + p.at * (a.D / 32);
    reinterpret_cast<uint32_t*>(codes)[lane] = code;
    if ((lane & 3) == 0) scales[lane >> 2] = (uint8_t)byte;
  }
}

template <class E, int N>
__global__ __launch_bounds__(kThreads) void read_kernel(RowsArgs a, int row_threads_shift) {
  const int w = blockIdx.y, lane = threadIdx.x & ((1 << row_threads_shift) - 1), size = 1 << a.page_shift;
  int64_t out[N];
  uint32_t code[N], scale[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    int t, h;
    out[i] = -1;
    code[i] = scale[i] = 0;
    if (token_head(a, ((blockIdx.x * N + i) * (uint32_t)kThreads + threadIdx.x) >> row_threads_shift, t, h)) {
      out[i] = ((int64_t)t * a.heads + h) * a.D + 8 * lane;
      const int slot = a.slots[t];
      if (slot >= 0 && slot < a.slot_count) {
        const Place p = place(a, slot, h);
        code[i] = reinterpret_cast<const uint32_t*>(p.page + (w ? size * (a.D / 2) : 0) + p.at * (a.D / 2))[lane];
        scale[i] = p.page[size * a.D + (w ? size * (a.D / 32) : 0) + p.at * (a.D / 32) + (lane >> 2)];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (out[i] >= 0) st8(static_cast<E*>(w ? a.v_out : a.k_out) + out[i], kv4_values<E>(code[i], kv4_scale(scale[i])));
}

}  // namespace

// N rows a thread where that leaves 1024 workgroups (4 a CU)
template <class F1, class F4>
void launch_rows(const RowsArgs& a, F1 one, F4 four) {
  const int shift = __builtin_ctz(a.D / 8);
  const int64_t blocks = (((int64_t)(a.T + 15) / 16 * 16 * a.heads << shift) + kThreads - 1) / kThreads;
  if (blocks >= 2048)
    four(dim3((unsigned)((blocks + 3) / 4), 2), shift);
  else
    one(dim3((unsigned)blocks, 2), shift);
}

void launch_kv4_write(const RowsArgs& a, hipStream_t st) {
  if (a.fp16)
    launch_rows(a, [&](dim3 grid, int shift) { write_kernel<f16, 1><<<grid, kThreads, 0, st>>>(a, shift); },
                [&](dim3 grid, int shift) { write_kernel<f16, 4><<<grid, kThreads, 0, st>>>(a, shift); });
  else
    launch_rows(a, [&](dim3 grid, int shift) { write_kernel<bf16, 1><<<grid, kThreads, 0, st>>>(a, shift); },
                [&](dim3 grid, int shift) { write_kernel<bf16, 4><<<grid, kThreads, 0, st>>>(a, shift); });
}

void launch_kv4_read(const RowsArgs& a, hipStream_t st) {
  if (a.fp16)
    launch_rows(a, [&](dim3 grid, int shift) { read_kernel<f16, 1><<<grid, kThreads, 0, st>>>(a, shift); },
                [&](dim3 grid, int shift) { read_kernel<f16, 4><<<grid, kThreads, 0, st>>>(a, shift); });
  else
    launch_rows(a, [&](dim3 grid, int shift) { read_kernel<bf16, 1><<<grid, kThreads, 0, st>>>(a, shift); },
                [&](dim3 grid, int shift) { read_kernel<bf16, 4><<<grid, kThreads, 0, st>>>(a, shift); });
}

}  // namespace cqgdn
