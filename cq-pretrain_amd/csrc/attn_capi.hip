// extern "C" entry points of the attention layers' operators (declared in include/cqgdn.h).
#include <hip/hip_runtime.h>

#include "attn_kernels.hpp"
#include "cqgdn.h"

using namespace cqgdn;

namespace {

int check_launch(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(CQGDN_EHIP, "%s: %s", what, hipGetErrorString(e));
  return ok();
}

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

bool page_ok(int page) { return page >= 16 && page <= 65536 && (page & (page - 1)) == 0; }
bool dim_ok(int D) { return D == 64 || D == 128 || D == 256; }

constexpr int64_t kThreads = 0x7FFFFFFF;  // threads of a launch

int check_cache(const void* data, int64_t pages, int kv_heads, int D, int page) {
  if (!dim_ok(D)) return fail(CQGDN_EUNSUPPORTED, "head_dim=%d: the 4-bit cache takes 64, 128 and 256", D);
  if (!page_ok(page)) return fail(CQGDN_EINVAL, "page=%d must be a power of two from 16 to 65536", page);
  if (kv_heads <= 0 || pages < 0) return fail(CQGDN_EINVAL, "invalid sizes pages=%lld kv_heads=%d", (long long)pages, kv_heads);
  if (pages * page > INT32_MAX)
    return fail(CQGDN_EUNSUPPORTED, "%lld pages of %d tokens: slots are 32-bit", (long long)pages, page);
  if (pages > 0 && (!data || !aligned(data, 16))) return fail(CQGDN_EINVAL, "data must be non-null and 16-byte aligned");
  return CQGDN_OK;
}

int check_rows(const char* what, int64_t T, int kv_heads, int D) {
  if (T < 0) return fail(CQGDN_EINVAL, "%s: T=%lld", what, (long long)T);
  if (T > kThreads / (D / 8) / kv_heads - 16)
    return fail(CQGDN_EUNSUPPORTED, "%s: T=%lld rows of %d heads are too many", what, (long long)T, kv_heads);
  return CQGDN_OK;
}

// the rows of one request that a launch is made for: the caller's bound, and no fewer than the requests have on
// average, so that a bound far too small costs neither workspace (parts of many rows) nor time
int row_bound(int64_t T, int N, int max_queries) {
  const int64_t bound = max_queries < T ? max_queries : T, average = N > 0 ? T / N : 1;
  return (int)(bound > average ? bound : average);
}

}  // namespace

extern "C" {

int cqgdn_rotary(const void* q, int64_t q_token, int64_t q_head, int q_heads, const void* k, int64_t k_token,
                 int64_t k_head, int k_heads, int64_t T, int head_dim, int rotary_dim, int adjacent, int backward,
                 int dtype, const void* positions, int wide_positions, int64_t axis_stride, int axes,
                 const uint64_t* turns, const int32_t* axis, void* q_out, void* k_out, void* stream) {
  if (T < 0 || q_heads < 0 || k_heads < 0 || head_dim <= 0 || head_dim % 2 || rotary_dim < 0 || rotary_dim % 2 ||
      rotary_dim > head_dim || axes <= 0)
    return fail(CQGDN_EINVAL, "invalid sizes T=%lld q_heads=%d k_heads=%d head_dim=%d rotary_dim=%d axes=%d",
                (long long)T, q_heads, k_heads, head_dim, rotary_dim, axes);
  if (dtype != CQGDN_BF16 && dtype != CQGDN_F16 && dtype != CQGDN_F32)
    return fail(CQGDN_EINVAL, "dtype=%d must be CQGDN_BF16, CQGDN_F16 or CQGDN_F32", dtype);
  if (q_heads > 65535 || k_heads > 65535 - q_heads)
    return fail(CQGDN_EUNSUPPORTED, "%d and %d heads are too many", q_heads, k_heads);
  if (T == 0 || q_heads + k_heads == 0) return ok();
  if ((q_heads > 0 && (!q || !q_out)) || (k_heads > 0 && (!k || !k_out)) || !positions ||
      (rotary_dim > 0 && (!turns || !axis)))
    return fail(CQGDN_EINVAL, "q, k, their outputs, positions, turns and axis must be non-null");
  if (T >= 1 << 24) return fail(CQGDN_EUNSUPPORTED, "T=%lld tokens are too many", (long long)T);
  const RotaryArgs a{{q, k}, {q_out, k_out}, {q_token, k_token}, {q_head, k_head}, {q_heads, k_heads}, T, head_dim,
                     rotary_dim, adjacent != 0, backward != 0, dtype, positions, wide_positions != 0, axis_stride,
                     axes, turns, axis};
  launch_rotary(a, (hipStream_t)stream);
  return check_launch("cqgdn_rotary");
}

int cqgdn_step_pages(const int32_t* cached, const int32_t* fresh, int N, int32_t* tables, int64_t table_stride,
                     int columns, int32_t* pool, int pool_size, const int32_t* pool_count, int page, int64_t T,
                     int32_t* starts, int32_t* lengths, int32_t* admitted, int32_t* count, int32_t* slots,
                     int32_t* positions, int32_t* visible, void* stream) {
  if (N < 0 || columns < 0 || pool_size < 0 || T < 0 || table_stride < columns)
    return fail(CQGDN_EINVAL, "invalid sizes N=%d columns=%d (stride %lld) pool=%d T=%lld", N, columns,
                (long long)table_stride, pool_size, (long long)T);
  if (!page_ok(page)) return fail(CQGDN_EINVAL, "page=%d must be a power of two from 16 to 65536", page);
  if ((int64_t)N * columns > INT32_MAX || T > INT32_MAX - 1024 || (int64_t)pool_size * page > INT32_MAX)
    return fail(CQGDN_EUNSUPPORTED, "N=%d columns=%d pool=%d T=%lld: counts and slots are 32-bit", N, columns,
                pool_size, (long long)T);
  if ((N > 0 && (!cached || !fresh || !lengths || !admitted)) || (N > 0 && columns > 0 && !tables) ||
      (pool_size > 0 && !pool) || !pool_count || !starts || !count || (T > 0 && (!slots || !positions || !visible)))
    return fail(CQGDN_EINVAL, "null buffer");
  const PagesArgs a{cached, fresh, N, tables, table_stride, columns, pool, pool_size, pool_count, __builtin_ctz(page),
                    (int)T, starts, lengths, admitted, count, slots, positions, visible};
  launch_pages(a, (hipStream_t)stream);
  return check_launch("cqgdn_step_pages");
}

size_t cqgdn_kv4_page_bytes(int page, int head_dim) {
  return page_ok(page) && dim_ok(head_dim) ? (size_t)kv4_page_bytes(page, head_dim) : 0;
}

int cqgdn_kv4_write(const void* k, int64_t k_token, int64_t k_head, const void* v, int64_t v_token, int64_t v_head,
                    int dtype, const int32_t* slots, int64_t T, int kv_heads, int head_dim, void* data, int64_t pages,
                    int page, void* stream) {
  if (const int e = check_cache(data, pages, kv_heads, head_dim, page)) return e;
  if (const int e = check_rows("cqgdn_kv4_write", T, kv_heads, head_dim)) return e;
  if (dtype != CQGDN_BF16 && dtype != CQGDN_F16) return fail(CQGDN_EINVAL, "dtype=%d must be CQGDN_BF16 or CQGDN_F16", dtype);
  if (T == 0 || pages == 0) return ok();
  if (!k || !v || !slots || !aligned(k, 16) || !aligned(v, 16) || k_token % 8 || k_head % 8 || v_token % 8 || v_head % 8)
    return fail(CQGDN_EINVAL, "k and v (16-byte aligned, strides multiples of 8 elements) and slots must be non-null");
  const RowsArgs a{k, v, {k_token, v_token}, {k_head, v_head}, nullptr, nullptr, slots, (int)T, kv_heads,
                   head_dim, static_cast<uint8_t*>(data), (int)(pages * page), __builtin_ctz(page), dtype == CQGDN_F16,
                   Divider(kv_heads)};
  launch_kv4_write(a, (hipStream_t)stream);
  return check_launch("cqgdn_kv4_write");
}

int cqgdn_kv4_read(const void* data, int64_t pages, int page, int kv_heads, int head_dim, const int32_t* slots,
                   int64_t T, int dtype, void* k, void* v, void* stream) {
  if (const int e = check_cache(data, pages, kv_heads, head_dim, page)) return e;
  if (const int e = check_rows("cqgdn_kv4_read", T, kv_heads, head_dim)) return e;
  if (dtype != CQGDN_BF16 && dtype != CQGDN_F16) return fail(CQGDN_EINVAL, "dtype=%d must be CQGDN_BF16 or CQGDN_F16", dtype);
  if (T == 0) return ok();
  if (!k || !v || !slots || !aligned(k, 16) || !aligned(v, 16))
    return fail(CQGDN_EINVAL, "k, v (16-byte aligned) and slots must be non-null");
  const RowsArgs a{nullptr, nullptr, {0, 0}, {0, 0}, k, v, slots, (int)T, kv_heads, head_dim,
                   static_cast<uint8_t*>(const_cast<void*>(data)), (int)(pages * page), __builtin_ctz(page),
                   dtype == CQGDN_F16, Divider(kv_heads)};
  launch_kv4_read(a, (hipStream_t)stream);
  return check_launch("cqgdn_kv4_read");
}

size_t cqgdn_kv4_attend_workspace_size(int64_t T, int N, int heads, int kv_heads, int head_dim, int max_queries,
                                       int columns, int page) {
  if (T <= 0 || N < 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads || !dim_ok(head_dim) || max_queries <= 0 ||
      columns < 0 || !page_ok(page))
    return 0;
  return attend_workspace_bytes(T, N, heads, kv_heads, head_dim, row_bound(T, N, max_queries), (int64_t)columns * page);
}

int cqgdn_kv4_attend(const void* q, int64_t q_token, int64_t q_head, int dtype, int64_t T, int heads, int head_dim,
                     const void* data, int64_t pages, int page, int kv_heads, const int32_t* tables,
                     int64_t table_stride, int columns, const int32_t* starts, int N, const int32_t* visible,
                     int window, float scale, int max_queries, void* out, float* lse, void* workspace,
                     size_t workspace_bytes, void* stream) {
  if (const int e = check_cache(data, pages, kv_heads, head_dim, page)) return e;
  if (dtype != CQGDN_BF16 && dtype != CQGDN_F16) return fail(CQGDN_EINVAL, "dtype=%d must be CQGDN_BF16 or CQGDN_F16", dtype);
  if (T < 0 || N < 0 || columns < 0 || table_stride < columns || heads <= 0 || heads % kv_heads || window < 0 ||
      max_queries <= 0 || !(scale - scale == 0.f))
    return fail(CQGDN_EINVAL,
                "invalid sizes T=%lld N=%d columns=%d (stride %lld) heads=%d kv_heads=%d window=%d max_queries=%d "
                "scale=%g", (long long)T, N, columns, (long long)table_stride, heads, kv_heads, window, max_queries,
                (double)scale);
  if (T == 0) return ok();
  if (T > (1 << 27) / heads || N >= (1 << 23) / kv_heads || kv_heads > 65535)
    return fail(CQGDN_EUNSUPPORTED, "T=%lld rows of %d heads, or N=%d requests, are too many", (long long)T, heads, N);
  if (!q || !out || !visible || !starts || (N > 0 && columns > 0 && !tables) || !aligned(q, 16) || !aligned(out, 16) ||
      q_token % 8 || q_head % 8)
    return fail(CQGDN_EINVAL, "q and out (16-byte aligned, strides multiples of 8 elements), tables, starts and "
                "visible must be non-null");
  const int most = row_bound(T, N, max_queries);
  const size_t need = attend_workspace_bytes(T, N, heads, kv_heads, head_dim, most, (int64_t)columns * page);
  if (need > 0 && (!workspace || !aligned(workspace, 256) || workspace_bytes < need))
    return fail(CQGDN_EINVAL, "workspace must be 256-byte aligned and >= cqgdn_kv4_attend_workspace_size");
  const AttendArgs a{q, q_token, q_head, T, heads, kv_heads, head_dim, static_cast<const uint8_t*>(data), (uint32_t)pages,
                     __builtin_ctz(page), tables, table_stride, pages > 0 ? columns : 0, starts, visible, N, window,
                     scale, dtype == CQGDN_F16, most, out, lse, static_cast<float*>(workspace), Divider(heads / kv_heads)};
  launch_attend(a, (hipStream_t)stream);
  return check_launch("cqgdn_kv4_attend");
}

}  // extern "C"
