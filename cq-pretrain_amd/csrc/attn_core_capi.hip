// extern "C" entry points of the attention over 16-bit keys and values (declared in include/cqgdn.h).
#include <hip/hip_runtime.h>

#include "attn_kernels.hpp"
#include "attn_plan.hpp"
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
bool type_ok(int dtype) { return dtype == CQGDN_BF16 || dtype == CQGDN_F16; }
bool finite(float x) { return x - x == 0.f; }
// rows as the kernels read them: the offsets of 64 tokens, and of a token's heads, fit 32 bits
bool rows_ok(const void* p, int64_t token, int64_t head, int heads) {
  return p && aligned(p, 16) && token % 8 == 0 && head % 8 == 0 && token >= 0 && token < 1 << 24 && head >= 0 &&
         head <= ((1 << 29) - 1) / heads;
}

int check_cache16(const void* data, int64_t pages, int kv_heads, int D, int page) {
  if (!dim_ok(D)) return fail(CQGDN_EUNSUPPORTED, "head_dim=%d: the 16-bit cache takes 64, 128 and 256", D);
  if (!page_ok(page)) return fail(CQGDN_EINVAL, "page=%d must be a power of two from 16 to 65536", page);
  if (kv_heads <= 0 || pages < 0) return fail(CQGDN_EINVAL, "invalid sizes pages=%lld kv_heads=%d", (long long)pages, kv_heads);
  if (pages * page > INT32_MAX)
    return fail(CQGDN_EUNSUPPORTED, "%lld pages of %d tokens: slots are 32-bit", (long long)pages, page);
  if (pages > 0 && (!data || !aligned(data, 16))) return fail(CQGDN_EINVAL, "data must be non-null and 16-byte aligned");
  return CQGDN_OK;
}

int check_scores(int dtype, float scale, float cap) {
  if (!type_ok(dtype)) return fail(CQGDN_EINVAL, "dtype=%d must be CQGDN_BF16 or CQGDN_F16", dtype);
  // what the kernels hold of them: both, and their quotient, in units of log2 e
  if (!finite(2.f * 1.45f * scale) || !finite(2.f * 1.45f * cap) || cap < 0.f || (cap > 0.f && !finite(2.f * scale / cap * 1.45f)))
    return fail(CQGDN_EINVAL, "scale=%g and cap=%g must be finite, and so their quotient, the cap not negative", (double)scale,
                (double)cap);
  return CQGDN_OK;
}

// the rows of one request that a launch is made for: the caller's bound, and no fewer than the requests have on average
int row_bound(int64_t T, int N, int max_queries) {
  const int64_t bound = max_queries < T ? max_queries : T, average = N > 0 ? T / N : 1;
  return (int)(bound > average ? bound : average);
}

size_t part_bytes(int64_t T, int heads, int D, int splits) {
  return splits > 1 ? (size_t)T * heads * splits * (D + 2) * sizeof(float) : 0;
}

// sizes of packed rows
int check_packed(int64_t T, int64_t S, int heads, int kv_heads, int D, const float* slopes) {
  if (!dim_ok(D)) return fail(CQGDN_EUNSUPPORTED, "head_dim=%d: attention takes 64, 128 and 256", D);
  if (T < 0 || S < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads)
    return fail(CQGDN_EINVAL, "invalid sizes T=%lld S=%lld heads=%d kv_heads=%d", (long long)T, (long long)S, heads, kv_heads);
  if (T > (1 << 27) / heads || S > (1 << 27) / kv_heads || heads > 65535)
    return fail(CQGDN_EUNSUPPORTED, "T=%lld rows of %d heads, or S=%lld keys of %d, are too many", (long long)T, heads,
                (long long)S, kv_heads);
  if (slopes && S > 1 << 24)
    return fail(CQGDN_EUNSUPPORTED, "S=%lld keys: distances are counted in fp32, over 2^24 keys at most", (long long)S);
  return CQGDN_OK;
}

}  // namespace

extern "C" {

int cqgdn_kv16_append(const void* q, int64_t q_token, int64_t q_head, int q_heads, const void* k, int64_t k_token,
                      int64_t k_head, const void* v, int64_t v_token, int64_t v_head, int64_t T, int kv_heads,
                      int head_dim, int rotary_dim, int adjacent, int dtype, const void* positions, int wide_positions,
                      int64_t axis_stride, int axes, const uint64_t* turns, const int32_t* axis, const int32_t* slots,
                      void* q_out, void* data, int64_t pages, int page, void* stream) {
  if (const int e = check_cache16(data, pages, kv_heads, head_dim, page)) return e;
  if (!type_ok(dtype)) return fail(CQGDN_EINVAL, "dtype=%d must be CQGDN_BF16 or CQGDN_F16", dtype);
  if (T < 0 || q_heads < 0 || rotary_dim < 0 || rotary_dim % 2 || rotary_dim > head_dim || axes < 0 ||
      (rotary_dim > 0 && axes == 0))
    return fail(CQGDN_EINVAL, "invalid sizes T=%lld q_heads=%d rotary_dim=%d axes=%d", (long long)T, q_heads, rotary_dim, axes);
  if (q_heads > 65535 || kv_heads > 65535 / 2 - q_heads / 2 || T >= 1 << 24)
    return fail(CQGDN_EUNSUPPORTED, "T=%lld tokens, or %d and %d heads, are too many", (long long)T, q_heads, kv_heads);
  if (T == 0) return ok();
  if ((q_heads > 0 && (!q || !q_out)) || !k || !v || !slots || (rotary_dim > 0 && (!positions || !turns || !axis)))
    return fail(CQGDN_EINVAL, "q and its output, k, v, slots, positions, turns and axis must be non-null");
  AppendArgs a{{{q, k}, {q_out, nullptr}, {q_token, k_token}, {q_head, k_head}, {q_heads, kv_heads}, T, head_dim,
                rotary_dim, adjacent != 0, false, dtype, positions, wide_positions != 0, axis_stride, axes, turns, axis},
               v, v_token, v_head, slots, data, (int)(pages * page), __builtin_ctz(page)};
  launch_append(a, (hipStream_t)stream);
  return check_launch("cqgdn_kv16_append");
}

size_t cqgdn_kv16_attend_workspace_size(int64_t T, int N, int heads, int kv_heads, int head_dim, int max_queries,
                                        int columns, int page) {
  if (T <= 0 || N < 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads || !dim_ok(head_dim) || max_queries <= 0 ||
      columns < 0 || !page_ok(page))
    return 0;
  return part_bytes(T, heads, head_dim,
                    attend_plan(N, kv_heads, heads / kv_heads, head_dim, row_bound(T, N, max_queries),
                                (int64_t)columns * page, 0).splits);
}

int cqgdn_kv16_attend(const void* q, int64_t q_token, int64_t q_head, int dtype, int64_t T, int heads, int head_dim,
                      const void* data, int64_t pages, int page, int kv_heads, const int32_t* tables,
                      int64_t table_stride, int columns, const int32_t* starts, int N, const int32_t* visible,
                      int window, const int32_t* positions, float scale, float cap, const float* slopes,
                      int max_queries, void* out, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  if (const int e = check_cache16(data, pages, kv_heads, head_dim, page)) return e;
  if (const int e = check_scores(dtype, scale, cap)) return e;
  if (T < 0 || N < 0 || columns < 0 || table_stride < columns || heads <= 0 || heads % kv_heads || window < 0 ||
      max_queries <= 0)
    return fail(CQGDN_EINVAL,
                "invalid sizes T=%lld N=%d columns=%d (stride %lld) heads=%d kv_heads=%d window=%d max_queries=%d",
                (long long)T, N, columns, (long long)table_stride, heads, kv_heads, window, max_queries);
  if (T == 0) return ok();
  if (T > (1 << 27) / heads || N >= (1 << 23) / kv_heads || kv_heads > 65535)
    return fail(CQGDN_EUNSUPPORTED, "T=%lld rows of %d heads, or N=%d requests, are too many", (long long)T, heads, N);
  if (!q || !out || !visible || !starts || (N > 0 && columns > 0 && !tables) || !aligned(q, 16) || !aligned(out, 16) ||
      q_token % 8 || q_head % 8)
    return fail(CQGDN_EINVAL, "q and out (16-byte aligned, strides multiples of 8 elements), tables, starts and "
                "visible must be non-null");
  const int most = row_bound(T, N, max_queries), group = heads / kv_heads;
  const int64_t capacity = (int64_t)columns * page;
  const size_t need = cqgdn_kv16_attend_workspace_size(T, N, heads, kv_heads, head_dim, max_queries, columns, page);
  if (need > 0 && (!workspace || !aligned(workspace, 256) || workspace_bytes < need))
    return fail(CQGDN_EINVAL, "workspace must be 256-byte aligned and >= cqgdn_kv16_attend_workspace_size");
  const CoreArgs a{{q, q_token, q_head, T, heads, kv_heads, head_dim, static_cast<const uint8_t*>(data), (uint32_t)pages,
                    __builtin_ctz(page), tables, table_stride, pages > 0 ? columns : 0, starts, visible, N, window,
                    scale, dtype == CQGDN_F16, most, out, lse, static_cast<float*>(workspace), Divider(group)},
                   nullptr, nullptr, 0, 0, 0, 0, 0, nullptr, positions, cap, slopes};
  const AttendPlan p = attend_plan(N, kv_heads, group, head_dim, most, pages > 0 ? capacity : 0, window);
  if (p.tiles)
    launch_core(a, true, p.splits, (hipStream_t)stream);
  else
    launch_core_few(a, p.splits, p.per, (hipStream_t)stream);
  if (p.splits > 1) launch_attend_join(a, p.splits, (hipStream_t)stream);
  return check_launch("cqgdn_kv16_attend");
}

size_t cqgdn_attend_fwd_workspace_size(int64_t T, int64_t S, int heads, int kv_heads, int head_dim) {
  if (T <= 0 || S < 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads || !dim_ok(head_dim)) return 0;
  return part_bytes(T, heads, head_dim, core_parts(T, S, heads, kv_heads, head_dim));
}

int cqgdn_attend_fwd(const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token, int64_t k_head,
                     const void* v, int64_t v_token, int64_t v_head, int dtype, int64_t T, int64_t S, int heads,
                     int kv_heads, int head_dim, const int32_t* first, const int32_t* limit, const int32_t* positions,
                     float scale, float cap, const float* slopes, void* out, float* lse, void* workspace,
                     size_t workspace_bytes, void* stream) {
  if (const int e = check_packed(T, S, heads, kv_heads, head_dim, slopes)) return e;
  if (const int e = check_scores(dtype, scale, cap)) return e;
  if (T == 0) return ok();
  if (!rows_ok(q, q_token, q_head, heads) ||
      (S > 0 && (!rows_ok(k, k_token, k_head, kv_heads) || !rows_ok(v, v_token, v_head, kv_heads))) || !limit || !out ||
      !aligned(out, 16))
    return fail(CQGDN_EINVAL, "q, k, v and out (16-byte aligned, strides multiples of 8 elements, not negative, below 2^24 "
                "a token and 2^29 all heads) and limit must be non-null");
  const int splits = core_parts(T, S, heads, kv_heads, head_dim);
  const size_t need = part_bytes(T, heads, head_dim, splits);
  if (need > 0 && (!workspace || !aligned(workspace, 256) || workspace_bytes < need))
    return fail(CQGDN_EINVAL, "workspace must be 256-byte aligned and >= cqgdn_attend_fwd_workspace_size");
  const CoreArgs a{{q, q_token, q_head, T, heads, kv_heads, head_dim, nullptr, 0, 0, nullptr, 0, 0, nullptr, limit, 1, 0,
                    scale, dtype == CQGDN_F16, (int)T, out, lse, static_cast<float*>(workspace), Divider(heads / kv_heads)},
                   k, v, k_token, k_head, v_token, v_head, (int)S, first, positions, cap, slopes};
  launch_core(a, false, splits, (hipStream_t)stream);
  if (splits > 1) launch_attend_join(a, splits, (hipStream_t)stream);
  return check_launch("cqgdn_attend_fwd");
}

size_t cqgdn_attend_bwd_workspace_size(int64_t T, int64_t S, int heads, int kv_heads, int head_dim) {
  if (T < 0 || S < 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads || !dim_ok(head_dim)) return 0;
  return core_backward_bytes(T, S, heads, kv_heads, head_dim);
}

int cqgdn_attend_bwd(const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token, int64_t k_head,
                     const void* v, int64_t v_token, int64_t v_head, const void* dy, int64_t dy_token, int64_t dy_head,
                     int dtype, int64_t T, int64_t S, int heads, int kv_heads, int head_dim, const int32_t* first,
                     const int32_t* limit, const int32_t* positions, float scale, float cap, const float* slopes,
                     const void* out, const float* lse, const float* dlse, void* dq, void* dk, void* dv,
                     void* workspace, size_t workspace_bytes, void* stream) {
  if (const int e = check_packed(T, S, heads, kv_heads, head_dim, slopes)) return e;
  if (const int e = check_scores(dtype, scale, cap)) return e;
  if (T == 0 && S == 0) return ok();
  if ((T > 0 && (!rows_ok(q, q_token, q_head, heads) || !rows_ok(dy, dy_token, dy_head, heads) || !limit || !out ||
                 !aligned(out, 16) || !lse || !dq || !aligned(dq, 16))) ||
      (S > 0 && (!rows_ok(k, k_token, k_head, kv_heads) || !rows_ok(v, v_token, v_head, kv_heads) || !dk != !dv ||
                 !aligned(dk, 16) || !aligned(dv, 16))))
    return fail(CQGDN_EINVAL, "q, k, v, dy, out and the gradients (16-byte aligned, strides multiples of 8 elements, "
                "not negative, below 2^24 a token and 2^29 all heads), limit and lse must be non-null");
  const size_t need = core_backward_bytes(T, S, heads, kv_heads, head_dim);
  if (need > 0 && (!workspace || !aligned(workspace, 256) || workspace_bytes < need))
    return fail(CQGDN_EINVAL, "workspace must be 256-byte aligned and >= cqgdn_attend_bwd_workspace_size");
  const CoreGradArgs a{{{q, q_token, q_head, T, heads, kv_heads, head_dim, nullptr, 0, 0, nullptr, 0, 0, nullptr, limit, 1, 0,
                         scale, dtype == CQGDN_F16, (int)T, nullptr, const_cast<float*>(lse), static_cast<float*>(workspace),
                         Divider(heads / kv_heads)},
                        k, v, k_token, k_head, v_token, v_head, (int)S, first, positions, cap, slopes},
                       dy, dy_token, dy_head, dlse, dq, dk, dv, nullptr, nullptr};
  launch_core_backward(a, (hipStream_t)stream);
  return check_launch("cqgdn_attend_bwd");
}

}  // extern "C"
