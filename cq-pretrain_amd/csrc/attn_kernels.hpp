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

// Rows put into the 16-bit pages: queries and keys turned, queries out as rotary has them.
struct AppendArgs : RotaryArgs {
  const void* v;
  int64_t v_token, v_head;
  const int32_t* slots;
  void* data;                  // [pages][kv_heads][2][page][D]
  int slot_count, page_shift;
};
void launch_append(const AppendArgs& a, hipStream_t st);

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
// adds up the parts of a call
void launch_attend_join(const AttendArgs& a, int splits, hipStream_t st);

// Attention over 16-bit keys and values: rows of packed documents, or the pages of a 16-bit cache.  Row t sees the
// keys [first[t], limit[t]) of the rows, or the positions [limit[t] - window, limit[t]) of its request's pages.
struct CoreArgs : AttendArgs {
  const void *k, *v;           // rows [S][kv_heads][D], or the pages [pages][kv_heads][2][page][D] in `data`
  int64_t k_token, k_head, v_token, v_head;
  int S;
  const int32_t* first;        // or null: from 0
  const int32_t* positions;    // where row t stands, for the bias; null: at its last key
  float cap;                   // 0: none
  const float* slopes;         // [heads], or null
};
// many rows, over packed rows or (paged) the pages; with more than one split its parts are joined by the caller
void launch_core(const CoreArgs& a, bool paged, int splits, hipStream_t st);
// few rows a request, over the pages, in `splits` parts of `per` steps of 64 positions
void launch_core_few(const CoreArgs& a, int splits, int per, hipStream_t st);

// Its gradients, over packed rows; `lse` is read, `ws` is core_backward_bytes() bytes.
struct CoreGradArgs : CoreArgs {
  const void* dy;              // the output's gradient, strides in elements
  int64_t dy_token, dy_head;
  const float* dlse;           // [T][heads], or null
  void *dq, *dk, *dv;          // dense
  void *ranges, *blocks;       // in the workspace: RowRange and RowBlock of each 64 rows
};
size_t core_backward_bytes(int64_t T, int64_t S, int heads, int kv_heads, int D);
void launch_core_backward(const CoreGradArgs& a, hipStream_t st);

}  // namespace cqgdn
