// The pages of a step: block tables, slot maps and row limits from request lengths, in one launch
// (two above kOneLaunch tokens).  Whole numbers, prefix sums over the requests:
//   starts  = sum of the new tokens before a request;
//   pages of finished requests go on top of the pool, in order;
//   a request that fits its table row and the step's buffer takes ceil((cached + new) / page) -
//   ceil(cached / page) pages from the top of the pool, in order; where the pool is too small for it,
//   it is not admitted (and, its need being counted, neither is a later one that needs pages).
// One workgroup scans the requests, so the state (pool, tables, counts) has one writer and the result
// does not depend on timing.
#include <hip/hip_runtime.h>

#include "attn_kernels.hpp"

namespace cqgdn {
namespace {

constexpr int kThreads = 1024;
constexpr int kOneLaunch = 4096;  // tokens that the scanning workgroup writes itself

// exclusive prefix sum over the workgroup; total is the sum over all its threads
template <class I>
__device__ __forceinline__ I scan(I x, int64_t* shared, I& total) {
  I* const part = reinterpret_cast<I*>(shared);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  I y = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const I z = __shfl_up(y, o, 64);
    if (lane >= o) y += z;
  }
  __syncthreads();  // part is free again
  if (lane == 63) part[wave] = y;
  __syncthreads();
  I before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    if (w < wave) before += part[w];
    total += part[w];
  }
  return before + y - x;
}

// the last r in 0 .. n - 1 with prefix[r] <= i, for prefix[0] = 0 <= i < prefix[n]
__device__ __forceinline__ int owner(const int32_t* prefix, int n, int i) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] <= i)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

__device__ __forceinline__ void token(const PagesArgs& a, int t, int total) {
  int p = 0, slot = -1;
  if (t < total) {
    const int r = owner(a.starts, a.N, t);
    const bool in = a.admitted[r] != 0;
    p = a.lengths[r] - (in ? a.fresh[r] : 0) + t - a.starts[r];
    if (in) {
      const int entry = a.tables[r * a.table_stride + (p >> a.page_shift)];
      const int64_t s = ((int64_t)entry << a.page_shift) + (p & ((1 << a.page_shift) - 1));
      if (entry >= 0 && s <= INT32_MAX) slot = (int)s;
    }
  }
  a.slots[t] = slot;
  a.positions[t] = p;
  a.visible[t] = slot >= 0 ? p + 1 : 0;
}

__global__ __launch_bounds__(kThreads) void pages_kernel(PagesArgs a) {
  __shared__ int64_t part[kThreads / 64];
  const int tid = threadIdx.x, up = (1 << a.page_shift) - 1, sh = a.page_shift;
  const int64_t room = (int64_t)a.columns << sh;
  const int count0 = min(max(*a.pool_count, 0), a.pool_size);
  int64_t tokens = 0;  // sums over the requests before this chunk; any lengths' sum fits 64 bits
  int gone = 0;
  for (int r0 = 0; r0 < a.N; r0 += kThreads) {
    const int r = r0 + tid;
    const int m = r < a.N ? a.fresh[r] : 0, c = r < a.N ? max(a.cached[r], 0) : 0;
    int64_t every;
    const int64_t s = tokens + scan<int64_t>(max(m, 0), part, every);
    if (r < a.N) a.starts[r] = (int)min(s, (int64_t)INT32_MAX);
    tokens += every;
    int all;
    const int freed = m < 0 ? (int)min(((int64_t)c + up) >> sh, (int64_t)a.columns) : 0;
    const int f = scan(freed, part, all);
    for (int j = 0; j < freed; ++j) {
      const int at = count0 + gone + f + j;
      if (at < a.pool_size) a.pool[at] = a.tables[r * a.table_stride + j];
    }
    gone += all;
  }
  if (tid == 0) a.starts[a.N] = (int)min(tokens, (int64_t)INT32_MAX);
  const int count = min(count0 + gone, a.pool_size);
  __syncthreads();  // the pool's new top and the starts are there for every thread
  int need = 0, taken = 0;
  for (int r0 = 0; r0 < a.N; r0 += kThreads) {
    const int r = r0 + tid;
    const int m = r < a.N ? a.fresh[r] : 0, c = r < a.N ? max(a.cached[r], 0) : 0;
    const bool fits = m > 0 && (int64_t)c + m <= room && (int64_t)a.starts[min(r, a.N)] + m <= a.T;
    const int first = (int)(((int64_t)c + up) >> sh);
    const int mine = fits ? (int)(((int64_t)c + m + up) >> sh) - first : 0;
    int all;
    const int o = need + scan(mine, part, all);
    need += all;
    const bool in = m <= 0 || (fits && (mine == 0 || o + mine <= count));
    if (r < a.N) {
      if (in)
        for (int j = 0; j < mine; ++j) a.tables[r * a.table_stride + first + j] = a.pool[count - 1 - o - j];
      a.lengths[r] = m < 0 ? 0 : c + (in ? m : 0);
      a.admitted[r] = in;
    }
    scan(in ? mine : 0, part, all);
    taken += all;
  }
  if (tid == 0) *a.count = count - taken;
  if (a.T > kOneLaunch) return;
  __syncthreads();
  for (int t = tid; t < a.T; t += kThreads) token(a, t, (int)min(tokens, (int64_t)a.T));
}

__global__ __launch_bounds__(256) void tokens_kernel(PagesArgs a) {
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t < a.T) token(a, t, min(a.starts[a.N], a.T));
}

}  // namespace

void launch_pages(const PagesArgs& a, hipStream_t st) {
  pages_kernel<<<1, kThreads, 0, st>>>(a);
  if (a.T > kOneLaunch) tokens_kernel<<<(a.T + 255) / 256, 256, 0, st>>>(a);
}

}  // namespace cqgdn
