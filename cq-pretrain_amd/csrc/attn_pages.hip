// The pages of a step: block tables, slot maps and row limits from request lengths, in one launch
// (two above kOneLaunch tokens).  Whole numbers, prefix sums over the requests:
//   starts  = sum of the new tokens before a request;
//   pages of finished requests go on top of the pool, in order;
//   a request that fits its table row and the step's buffer takes ceil((cached + new) / page) -
//   ceil(cached / page) pages from the top of the pool, in order; where the pool is too small for it,
//   it is not admitted (and, its need being counted, neither is a later one that needs pages).
// One workgroup scans the requests, so the state (pool, tables, counts) has one writer and the result
// does not depend on timing.  A prefix sum gives every page that moves, and every row, its request by a binary
// search, so that all 1024 threads move them whatever the requests' sizes (64 requests, some of which return a
// hundred pages: 15 us one after the other, 6.6 like this): what is left is the latency of some six dependent rounds
// of memory and of the scans.  1000 requests: 10.6 us, and 4.6 for 28 thousand rows.
#include <hip/hip_runtime.h>

#include "attn_kernels.hpp"

namespace cqgdn {
namespace {

constexpr int kThreads = 1024;    // and requests of a round
constexpr int kOneLaunch = 4096;  // rows that the scanning workgroup writes itself

// exclusive prefix sums over the workgroup of x and y; sx and sy become the sums over all its threads
struct Parts {
  int64_t x[kThreads / 64];
  int y[kThreads / 64];
};
__device__ __forceinline__ void scan(int64_t& x, int& y, int64_t& sx, int& sy, Parts& part) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t x0 = x;
  const int y0 = y;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t p = __shfl_up(x, o, 64);
    const int q = __shfl_up(y, o, 64);
    if (lane >= o) {
      x += p;
      y += q;
    }
  }
  __syncthreads();  // part is free again
  if (lane == 63) {
    part.x[wave] = x;
    part.y[wave] = y;
  }
  __syncthreads();
  sx = 0;
  sy = 0;
  int64_t bx = 0;
  int by = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    if (w < wave) {
      bx += part.x[w];
      by += part.y[w];
    }
    sx += part.x[w];
    sy += part.y[w];
  }
  x += bx - x0;
  y += by - y0;
}

// the last r in 0 .. n - 1 with prefix[r] <= i, for prefix[0] <= i
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

// row t, at position p of request r
__device__ __forceinline__ void row(const PagesArgs& a, int t, int r, int p, bool in) {
  int slot = -1;
  if (in) {
    const int entry = a.tables[r * a.table_stride + (p >> a.page_shift)];
    const int64_t s = ((int64_t)entry << a.page_shift) + (p & ((1 << a.page_shift) - 1));
    if (entry >= 0 && s <= INT32_MAX) slot = (int)s;
  }
  a.slots[t] = slot;
  a.positions[t] = p;
  a.visible[t] = slot >= 0 ? p + 1 : 0;
}

__global__ __launch_bounds__(kThreads) void pages_kernel(PagesArgs a) {
  __shared__ Parts part;
  __shared__ int32_t prefix[kThreads], start[kThreads], base[kThreads];
  __shared__ bool admitted[kThreads];
  __shared__ int taken;
  const int tid = threadIdx.x, up = (1 << a.page_shift) - 1, sh = a.page_shift;
  const int64_t room = (int64_t)a.columns << sh;
  const int count0 = min(max(*a.pool_count, 0), a.pool_size);
  const bool once = a.N <= kThreads;  // one round: its values stay in registers and LDS
  if (tid == 0) taken = 0;
  int m = 0, c = 0;
  int64_t first_row = 0, tokens = 0;  // rows before the thread's request, and before the round's; 64 bits hold any
  const auto request = [&](int r) {
    m = r < a.N ? a.fresh[r] : 0;
    c = r < a.N ? max(a.cached[r], 0) : 0;
  };
  int gone = 0;
  for (int r0 = 0; r0 < a.N; r0 += kThreads) {
    const int r = r0 + tid, n = min(kThreads, a.N - r0);
    request(r);
    const int freed = m < 0 ? (int)min(((int64_t)c + up) >> sh, (int64_t)a.columns) : 0;
    int64_t x = max(m, 0), every;
    int f = freed, all;
    scan(x, f, every, all, part);
    first_row = tokens + x;
    const int clamped = (int)min(first_row, (int64_t)INT32_MAX);
    prefix[tid] = f;
    start[tid] = clamped;
    if (r < a.N) a.starts[r] = clamped;
    tokens += every;
    if (all) {
      __syncthreads();
      for (int i = tid; i < all; i += kThreads) {
        const int o = owner(prefix, n, i), at = count0 + gone + i;
        if (at < a.pool_size) a.pool[at] = a.tables[(r0 + o) * a.table_stride + i - prefix[o]];
      }
      gone += all;
    }
  }
  if (tid == 0) a.starts[a.N] = (int)min(tokens, (int64_t)INT32_MAX);
  const int count = min(count0 + gone, a.pool_size);
  __syncthreads();  // the pool's new top and the starts are there for every thread
  int need = 0;
  for (int r0 = 0; r0 < a.N; r0 += kThreads) {
    const int r = r0 + tid, n = min(kThreads, a.N - r0);
    if (!once) {
      request(r);
      first_row = r < a.N ? a.starts[r] : 0;
    }
    const bool fits = m > 0 && (int64_t)c + m <= room && first_row + m <= a.T;
    const int held = (int)(((int64_t)c + up) >> sh);
    const int mine = fits ? (int)(((int64_t)c + m + up) >> sh) - held : 0;
    int64_t x = 0, none;
    int o = mine, all;
    scan(x, o, none, all, part);
    const bool in = m <= 0 || (fits && (mine == 0 || need + o + mine <= count));
    // those before the first that finds no pages take all they need
    if (in && mine > 0) atomicMax(&taken, need + o + mine);
    prefix[tid] = o;
    admitted[tid] = in;
    base[tid] = held;
    if (r < a.N) {
      a.lengths[r] = m < 0 ? 0 : c + (in ? m : 0);
      a.admitted[r] = in;
    }
    if (all) {
      __syncthreads();
      for (int i = tid; i < all; i += kThreads) {
        const int w = owner(prefix, n, i);
        if (admitted[w]) a.tables[(r0 + w) * a.table_stride + base[w] + i - prefix[w]] = a.pool[count - 1 - need - i];
      }
      need += all;
    }
  }
  __syncthreads();  // the tables and what was taken are there for every thread
  if (tid == 0) *a.count = count - taken;
  if (a.T > kOneLaunch) return;
  base[tid] = c;
  __syncthreads();
  const int total = (int)min(tokens, (int64_t)a.T);
  for (int t = tid; t < a.T; t += kThreads) {
    if (t >= total) {
      row(a, t, 0, 0, false);
    } else if (once) {
      const int r = owner(start, a.N, t);
      row(a, t, r, base[r] + t - start[r], admitted[r]);
    } else {
      const int r = owner(a.starts, a.N, t);
      const bool in = a.admitted[r] != 0;
      row(a, t, r, a.lengths[r] - (in ? a.fresh[r] : 0) + t - a.starts[r], in);
    }
  }
}

__global__ __launch_bounds__(256) void tokens_kernel(PagesArgs a) {
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= a.T) return;
  if (t >= min(a.starts[a.N], a.T)) {
    row(a, t, 0, 0, false);
    return;
  }
  const int r = owner(a.starts, a.N, t);
  const bool in = a.admitted[r] != 0;
  row(a, t, r, a.lengths[r] - (in ? a.fresh[r] : 0) + t - a.starts[r], in);
}

}  // namespace

void launch_pages(const PagesArgs& a, hipStream_t st) {
  pages_kernel<<<1, kThreads, 0, st>>>(a);
  if (a.T > kOneLaunch) tokens_kernel<<<(a.T + 255) / 256, 256, 0, st>>>(a);
}

}  // namespace cqgdn
