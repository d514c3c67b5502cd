// Argument blocks and launchers of the attention layers' kernels: rotary positions, the pages of the
// 4-bit cache, the rows written into them and read back, and the attention that reads them
// (internal to libcqgdn).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "gdn_timer.hpp"

namespace cqgdn {

// A page of the 4-bit cache, for one head: key codes [page][D/2], value codes [page][D/2], key scale
// bytes [page][D/32], value scale bytes [page][D/32].  A code is e2m1 (sign, two exponent bits, one
// mantissa bit: 0 .5 1 1.5 2 3 4 6), the even value of a pair in its byte's low half; a scale byte b
// multiplies 32 neighbouring values by 2^(b - 127), and 255 makes them NaN.  A power of two keeps the
// products exact in bf16, and the conversion instructions of gfx950 take codes and scale together.
__host__ __device__ constexpr int kv4_page_bytes(int page, int D) { return page * (D + D / 16); }

// Division of n < 2^31 by d > 0 as a product: m = ceil(2^(31 + s) / d) with 2^s >= d is off by less than
// 2^s / d / 2^(31 + s) of a unit, n times which stays below 1 / d.
struct Divider {
  uint32_t d, m;
  int s;
  explicit Divider(uint32_t by) : d(by), m(0), s(0) {
    while ((1ull << s) < by) ++s;
    m = (uint32_t)(((1ull << (31 + s)) + by - 1) / by);
  }
  __device__ __forceinline__ int of(int n) const { return s == 0 ? n : (int)(__umulhi((uint32_t)n, m) >> (s - 1)); }
};

struct RotaryArgs {
  const void* x[2];            // q, k
  void* y[2];
  int64_t token[2], head[2];   // strides of x in elements; y is dense [T][heads][D]
  int heads[2];
  int64_t T;
  int D, rotary;               // head dimension, values of it that turn
  bool adjacent, back;
  int dtype;                   // CQGDN_BF16, CQGDN_F16 or CQGDN_F32
  const void* positions;       // [axes][T], int32 or int64
  bool wide;                   // int64 positions
  int64_t axis_stride;
  int axes;
  const uint64_t* turns;       // [rotary / 2] turns a position, in units of 2^-64 of a turn
  const int32_t* axis;         // [rotary / 2]
  Divider by_heads{1}, by_pairs{1};  // set by the launch
};
void launch_rotary(const RotaryArgs& a, hipStream_t st);

struct PagesArgs {
  const int32_t *cached, *fresh;  // [N]
  int N;
  int32_t* tables;                // [N][columns]
  int64_t table_stride;
  int columns;
  int32_t* pool;
  int pool_size;
  const int32_t* pool_count;
  int page_shift;
  int T;
  int32_t *starts, *lengths, *admitted, *count, *slots, *positions, *visible;
};
void launch_pages(const PagesArgs& a, hipStream_t st);

struct RowsArgs {                 // rows written to, or read from, the cache
  const void *k, *v;
  int64_t token[2], head[2];
  void *k_out, *v_out;
  const int32_t* slots;
  int T, heads, D;
  uint8_t* data;
  int slot_count, page_shift;     // pages x page, which 31 bits hold
  bool fp16;
  Divider by_heads;
};
void launch_kv4_write(const RowsArgs& a, hipStream_t st);
void launch_kv4_read(const RowsArgs& a, hipStream_t st);

struct AttendArgs {
  const void* q;
  int64_t q_token, q_head;
  int64_t T;
  int heads, kv_heads, D;
  const uint8_t* data;
  uint32_t page_count;
  int page_shift;
  const int32_t* tables;
  int64_t table_stride;
  int columns;
  const int32_t *starts, *visible;
  int N, window;
  float scale;
  bool fp16;
  int max_queries;
  void* out;
  float* lse;
  float* ws;
  Divider group;               // heads / kv_heads
};
// bytes of a call's workspace: the parts' O, maxima and sums, where the positions are split
size_t attend_workspace_bytes(int64_t T, int64_t N, int heads, int kv_heads, int D, int max_queries, int64_t capacity);
void launch_attend(const AttendArgs& a, hipStream_t st);
// the kernel for many rows a request (attn_tile.hip); with more than one split its parts are joined by the caller
void launch_attend_tiles(const AttendArgs& a, int splits, hipStream_t st);

}  // namespace cqgdn
