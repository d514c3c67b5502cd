// Attention of a step's query rows over the 4-bit pages.
//
// Row (t, query head) sees the positions [max(0, visible - window), visible) of its request and gets
// sum_j p_j v_j / sum_j p_j with p_j = exp(scale q k_j - m), in one pass over the positions with the
// running maximum m.  Rows of one request and one key head (new tokens x query heads of the group) are
// the columns of S^T = K Q^T, 16 at a time, so a lane owns one row: its limits, maximum and sum are the
// lane's own, and S^T's layout is already the operand of O^T = V^T P^T.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attn_kernels.hpp"
#include "attn_kv4.hpp"

namespace cqgdn {
namespace {

constexpr int kWaves = 4;     // of a workgroup; they take its steps in turn
constexpr int kStep = 32;     // positions of a wave's step
constexpr int kMaxSplits = 64;
constexpr int kFewRows = 32;  // of a request and key head: more take the kernel of attn_tile.hip

// The pages of one step's two halves of 16 positions, the codes of its 32 keys and values, and their
// scale bytes.  Lane (r16, q4) holds key r16 of either half: 16 bytes from each 128 dimensions (8 where
// D is 64), which are one block of 32, so an MFMA step's K index (q4, j) stands for dimension
// 128 x + 32 q4 + 8 kk + j and Q is read likewise.  Values come in rows: 16 bytes (a block) a lane.
template <int D>
struct Codes {
  static constexpr int XK = D > 128 ? D / 128 : 1;  // key loads a half
  static constexpr int WK = D >= 128 ? 4 : 2;       // words of one
  static constexpr int NV = D / 64;                 // value loads of the step
  uint32_t k[2][XK][WK];
  uint8_t ks[2][XK];
  u32x4 v[NV];
  uint8_t vs[NV];
  bool ok[2];
};

template <int D>
__device__ __forceinline__ int value_token(int j, int lane) {
  constexpr int PV = D / 32;  // 16-byte pieces of a row
  return (j * 64 + lane) / PV;
}

template <int D>
__device__ __forceinline__ void load(const AttendArgs& a, Codes<D>& c, const int (&page)[2], int pos, int h, int lane) {
  const int r16 = lane & 15, q4 = lane >> 4, size = 1 << a.page_shift;
  const uint8_t* base[2];
  int at[2];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    c.ok[half] = page[half] >= 0 && page[half] < a.pages;  // an entry that names no page: its positions are hidden
    base[half] = a.data + ((int64_t)(c.ok[half] ? page[half] : 0) * a.kv_heads + h) * kv4_page_bytes(size, D);
    at[half] = (pos + 16 * half) & (size - 1);
#pragma unroll
    for (int x = 0; x < Codes<D>::XK; ++x) {
      const uint8_t* p = base[half] + (at[half] + r16) * (D / 2);
      const uint8_t* s = base[half] + size * D + (at[half] + r16) * (D / 32);
      if constexpr (D >= 128) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(p + 64 * x + 16 * q4);
#pragma unroll
        for (int i = 0; i < 4; ++i) c.k[half][x][i] = w[i];
        c.ks[half][x] = s[4 * x + q4];
      } else {
        const uint2 w = *reinterpret_cast<const uint2*>(p + 8 * q4);
        c.k[half][x][0] = w.x;
        c.k[half][x][1] = w.y;
        c.ks[half][x] = s[q4 >> 1];
      }
    }
  }
#pragma unroll
  for (int j = 0; j < Codes<D>::NV; ++j) {
    constexpr int PV = D / 32;
    const int tok = value_token<D>(j, lane), piece = lane % PV;
    const int half = D == 64 ? tok >> 4 : j * 64 / PV / 16;
    const uint8_t* b = half ? base[1] : base[0];
    const int row = (half ? at[1] : at[0]) + (tok & 15);
    c.v[j] = *reinterpret_cast<const u32x4*>(b + size * (D / 2) + row * (D / 2) + 16 * piece);
    c.vs[j] = b[size * D + size * (D / 32) + row * (D / 32) + piece];
  }
}

__device__ __forceinline__ int min16(int x) {
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) x = min(x, __shfl_xor(x, o, 64));
  return x;
}
__device__ __forceinline__ int max16(int x) {
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) x = max(x, __shfl_xor(x, o, 64));
  return x;
}

// One workgroup: 16 rows of one request and key head, one of `splits` parts of the positions.  The
// waves' steps interleave, each with its own maximum, sum and O^T, and are joined at the end.
template <class E, int D>
__global__ __launch_bounds__(64 * kWaves) void attend_kernel(AttendArgs a, int tiles, int splits) {
  typedef typename Vec<E>::x8 x8;
  constexpr int LD = D + 16;  // 8 banks further each row: the transposed reads of 8 rows meet no bank twice
  constexpr int KQ = D / 32, MT = D / 16;
  __shared__ __align__(16) E vt[kWaves][kStep * LD];
  __shared__ float wm[kWaves][16], wl[kWaves][16];
  static_assert(kStep * LD * sizeof(E) >= 16 * D * sizeof(float), "the waves' O^T pass through their value tiles");
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, q4 = lane >> 4;
  int b = blockIdx.x;
  const int s = b % splits;
  b /= splits;
  const int h = b % a.kv_heads;
  b /= a.kv_heads;
  const int tile0 = b % tiles, r = b / tiles, group = a.heads / a.kv_heads, T = (int)a.T;
  const int from = r == 0 ? 0 : min(max(a.starts[r], 0), T);
  const int to = r == a.N ? T : min(max(a.starts[r + 1], from), T);  // request N: the padding behind the last
  const int rows = (to - from) * group;
  const int room = (int)min((int64_t)a.columns << a.page_shift, (int64_t)INT32_MAX - 1024);

  for (int tile = tile0; tile * 16 < rows; tile += tiles) {
    const int rho = tile * 16 + r16;
    const bool real = rho < rows;
    const int t = from + (real ? rho / group : 0), head = h * group + (real ? rho % group : 0);
    const int hi = real && r < a.N ? min(max(a.visible[t], 0), room) : 0;
    const int lo = a.window > 0 ? max(0, hi - a.window) : 0;
    // over the rows that see anything: from the first position any of them sees to the last, and the
    // range that all of them see, where nothing is masked
    const int first = min16(hi > 0 ? lo : INT32_MAX), last = max16(hi);
    const int low = max16(lo), high = min16(real ? hi : INT32_MAX);

    x8 qf[KQ];
    {
      const E* q = static_cast<const E*>(a.q) + t * a.q_token + head * a.q_head;
#pragma unroll
      for (int i = 0; i < KQ; ++i)
        qf[i] = real ? ld8(q + (D >= 128 ? 128 * (i / 4) + 32 * q4 + 8 * (i % 4) : 16 * q4 + 8 * i)) : zero8v<E>();
    }
    f32x4 o[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) o[i] = zero4();
    float m = -INFINITY, l = 0.f;

    const int begin = last > 0 ? first & ~(kStep - 1) : 0;
    const int steps = (last - begin + kStep - 1) / kStep;
    const int per = (((steps + splits - 1) / splits) + kWaves - 1) / kWaves * kWaves;
    const int stop = min(steps, (s + 1) * per);
    const float c = a.scale * 1.44269504088896341f;
    E* const vw = vt[wave];

    int i = s * per + wave;
    if (i < stop) {
      Codes<D> next;
      int pg[2];
      {
        const int pos = begin + i * kStep;
        pg[0] = page_of(a, r, pos);
        pg[1] = page_of(a, r, pos + 16);
        load<D>(a, next, pg, pos, h, lane);
        pg[0] = page_of(a, r, pos + kWaves * kStep);
        pg[1] = page_of(a, r, pos + kWaves * kStep + 16);
      }
      for (; i < stop; i += kWaves) {
        const Codes<D> now = next;
        const int pos = begin + i * kStep;
        if (i + kWaves < stop) {
          load<D>(a, next, pg, pos + kWaves * kStep, h, lane);
          pg[0] = page_of(a, r, pos + 2 * kWaves * kStep);
          pg[1] = page_of(a, r, pos + 2 * kWaves * kStep + 16);
        }
        const bool full = pos >= low && pos + kStep <= high && now.ok[0] && now.ok[1];
        // scores, in units of log2
        float sc[8];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          f32x4 acc = zero4();
#pragma unroll
          for (int x = 0; x < Codes<D>::XK; ++x) {
            const float ks = kv4_scale(now.ks[half][x]);
#pragma unroll
            for (int w = 0; w < Codes<D>::WK; ++w)
              acc = mfma(kv4_values<E>(now.k[half][x][w], ks), qf[x * Codes<D>::WK + w], acc);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float y = acc[e] * c;
            if (!full) {
              const int p = pos + 16 * half + 4 * q4 + e;
              if (p < lo || p >= hi || !now.ok[half]) y = -INFINITY;
            }
            sc[4 * half + e] = y;
          }
        }
        float top = sc[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) top = fmaxf(top, sc[e]);
        if (__any(top > m + kLazy)) {  // the maximum moves rarely, and for each row by itself
          top = fmaxf(top, __shfl_xor(top, 16, 64));
          top = fmaxf(top, __shfl_xor(top, 32, 64));
          if (top > m + kLazy) {
            const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
            m = top;
            l *= f;
#pragma unroll
            for (int k = 0; k < MT; ++k) o[k] *= f;
          }
        }
        const float base = (m == -INFINITY ? 0.f : m) - kAttendBias<E>;
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          p[e] = __builtin_amdgcn_exp2f(sc[e] - base);
          l += p[e];
        }
        const x8 pf = to8<E>(f32x8{p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7]});
        // values, row by row; where not every row sees every position, a position that none sees is zero,
        // and a NaN reaches only the rows that see it
#pragma unroll
        for (int j = 0; j < Codes<D>::NV; ++j) {
          constexpr int PV = D / 32;
          const int tok = value_token<D>(j, lane), piece = lane % PV;
          u32x4 w = now.v[j];
          uint32_t sb = now.vs[j];
          if (!full) {
            const bool any = pos + tok >= first && pos + tok < last && ((tok >> 4) ? now.ok[1] : now.ok[0]);
            uint64_t bad = __ballot(any && sb == 255);
            if (!any || sb == 255) {
              w = u32x4{0, 0, 0, 0};
              sb = 0;
            }
            for (; bad; bad &= bad - 1) {
              const int n = __builtin_ctzll(bad), at = pos + value_token<D>(j, n);
              const float add = at >= lo && at < hi ? __builtin_nanf("") : 0.f;
#pragma unroll
              for (int k = 0; k < MT; ++k)
                if (k / 2 == n % PV) o[k] += add;
            }
          }
          const float vs = kv4_scale(sb);
#pragma unroll
          for (int e = 0; e < 4; ++e) st8(vw + tok * LD + 32 * piece + 8 * e, kv4_values<E>(w[e], vs));
        }
#pragma unroll
        for (int k = 0; k < MT; ++k) o[k] = mfma(ld8_trpv<E>(vw, LD, 0, 16 * k), pf, o[k]);
      }
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    // join the waves: O^T rows through LDS, their 16-byte columns XORed with the row against bank conflicts
    float* const ow = reinterpret_cast<float*>(vw);
#pragma unroll
    for (int k = 0; k < MT; ++k)
      *reinterpret_cast<f32x4*>(ow + r16 * D + 4 * ((4 * k + q4) ^ r16)) = o[k];
    if (q4 == 0) {
      wm[wave][r16] = m;
      wl[wave][r16] = l;
    }
    __syncthreads();
    {
      const int row = tid >> 4, n = tile * 16 + row;
      float M = wm[0][row];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) M = fmaxf(M, wm[w][row]);
      float f[kWaves], L = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        f[w] = wm[w][row] == -INFINITY ? 0.f : exp2f(wm[w][row] - M);
        L += f[w] * wl[w][row];
      }
      if (n < rows) {
        const int64_t at = (int64_t)(from + n / group) * a.heads + h * group + n % group;
        const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
        for (int k = 0; k < D / 64; ++k) {
          const int col = (tid & 15) + 16 * k;
          f32x4 y = zero4();
#pragma unroll
          for (int w = 0; w < kWaves; ++w)
            y += f[w] * *reinterpret_cast<const f32x4*>(reinterpret_cast<float*>(vt[w]) + row * D + 4 * (col ^ row));
          if (splits == 1)
            st4(static_cast<E*>(a.out) + at * D + 4 * col, L == 0.f ? zero4() : y * inv);
          else if (M != -INFINITY || L != 0.f)  // the join reads no part that saw nothing
            *reinterpret_cast<f32x4*>(a.ws + (at * splits + s) * D + 4 * col) = y;
        }
        if ((tid & 15) == 0) {
          if (splits > 1) {
            float* ml = a.ws + a.T * a.heads * splits * D + (at * splits + s) * 2;
            ml[0] = M;
            ml[1] = L;
          } else if (a.lse) {
            a.lse[at] = (M - kAttendBias<E> + log2f(L)) * 0.693147180559945309f;
          }
        }
      }
    }
    __syncthreads();
  }
}

// Joins the parts of a row: 16 rows a workgroup, 16 lanes a row.
template <class E, int D>
__global__ __launch_bounds__(256) void join_kernel(AttendArgs a, int splits) {
  const int64_t at = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  if (at >= a.T * a.heads) return;
  const float* ml = a.ws + a.T * a.heads * splits * D + at * splits * 2;
  float M = -INFINITY;
  for (int s = 0; s < splits; ++s) M = fmaxf(M, ml[2 * s]);
  float L = 0.f;
  f32x4 y[D / 64];
#pragma unroll
  for (int k = 0; k < D / 64; ++k) y[k] = zero4();
  for (int s = 0; s < splits; ++s) {
    if (ml[2 * s] == -INFINITY && ml[2 * s + 1] == 0.f) continue;
    const float f = exp2f(ml[2 * s] - M);
    L += f * ml[2 * s + 1];
#pragma unroll
    for (int k = 0; k < D / 64; ++k)
      y[k] += f * *reinterpret_cast<const f32x4*>(a.ws + (at * splits + s) * D + 4 * ((threadIdx.x & 15) + 16 * k));
  }
#pragma unroll
  for (int k = 0; k < D / 64; ++k)
    st4(static_cast<E*>(a.out) + at * D + 4 * ((threadIdx.x & 15) + 16 * k), L == 0.f ? zero4() : y[k] * (1.f / L));
  if (a.lse && (threadIdx.x & 15) == 0) a.lse[at] = (M - kAttendBias<E> + log2f(L)) * 0.693147180559945309f;
}

// How a call runs: by which kernel, and in how many parts of the positions.
struct Plan {
  bool tiles;
  int splits;
};
Plan attend_plan(int64_t N, int kv_heads, int group, int max_queries, int64_t capacity) {
  const int64_t rows = (int64_t)max_queries * group;
  if (rows > kFewRows) {
    const int64_t blocks = N * kv_heads * ((rows + 127) / 128), most = std::min<int64_t>(kMaxSplits, (capacity + 511) / 512);
    return {true, (int)std::max<int64_t>(1, std::min(most, 512 / std::max<int64_t>(blocks, 1)))};
  }
  // as many parts as bring 1024 workgroups (4 a CU), each of at least 128 positions
  const int64_t blocks = N * kv_heads * ((rows + 15) / 16), most = std::min<int64_t>(kMaxSplits, (capacity + 127) / 128);
  return {false, (int)std::max<int64_t>(1, std::min(most, 1024 / std::max<int64_t>(blocks, 1)))};
}

template <class E, int D>
void launch_dim(const AttendArgs& a, hipStream_t st) {
  const int group = a.heads / a.kv_heads;
  const Plan p = attend_plan(a.N, a.kv_heads, group, a.max_queries, (int64_t)a.columns << a.page_shift);
  if (p.tiles) {
    launch_attend_tiles(a, p.splits, st);
  } else {
    const int64_t each = (int64_t)(a.N + 1) * a.kv_heads * p.splits;
    const int tiles = (int)std::max<int64_t>(1, std::min<int64_t>(((int64_t)a.max_queries * group + 15) / 16, (1 << 23) / each));
    // a workgroup takes every tiles-th tile: none is left out whatever the bound
    attend_kernel<E, D><<<(unsigned)(each * tiles), 64 * kWaves, 0, st>>>(a, tiles, p.splits);
  }
  if (p.splits > 1) join_kernel<E, D><<<(unsigned)((a.T * a.heads + 15) / 16), 256, 0, st>>>(a, p.splits);
}

template <class E>
void by_dim(const AttendArgs& a, hipStream_t st) {
  if (a.D == 64)
    launch_dim<E, 64>(a, st);
  else if (a.D == 128)
    launch_dim<E, 128>(a, st);
  else
    launch_dim<E, 256>(a, st);
}

}  // namespace

size_t attend_workspace_bytes(int64_t T, int64_t N, int heads, int kv_heads, int D, int max_queries, int64_t capacity) {
  const int splits = attend_plan(N, kv_heads, heads / kv_heads, max_queries, capacity).splits;
  return splits > 1 ? (size_t)T * heads * splits * (D + 2) * sizeof(float) : 0;
}

void launch_attend(const AttendArgs& a, hipStream_t st) {
  if (a.fp16)
    by_dim<f16>(a, st);
  else
    by_dim<bf16>(a, st);
}

}  // namespace cqgdn
