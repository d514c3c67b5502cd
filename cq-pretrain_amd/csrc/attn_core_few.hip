// Attention of few rows a request over the pages of a 16-bit cache: decode steps.
//
// Rows of one request and key head (new tokens x query heads of the group) are the columns of S^T = K Q^T, 16 at a
// time, so a lane owns one row: its limits, maximum, sum and slope are the lane's own, and S^T's layout is already the
// operand of O^T = V^T P^T.  Keys go from memory to the registers that the MFMAs take them from; values pass through
// shared memory, which turns them.  Four waves a workgroup take 32 positions each in turn, with a maximum, sum and O^T
// of their own, and are joined at the end; a workgroup takes one of `splits` parts of the positions.
//
// Bound by memory: 64 requests of up to 8192 positions, 4 key heads of 128, 144 us, 4.5 TB/s (a large copy reaches 4.8); one
// request of 9216, in parts, 11 us, most of it the latency of one round of loads after another.
//
// Scores, sums and O are fp32, a weight is rounded once to the rows' type for its product with V.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attn_core.hpp"
#include "attn_plan.hpp"

namespace cqgdn {
namespace {

constexpr int kPadding = 16;  // workgroups a key head for rows behind the requests'
constexpr int kHalf = 32;     // positions that a wave loads at once

// over the 16 rows, by rotations of a row of lanes; the four rows hold the same
template <int N>
__device__ __forceinline__ int turned(int x) {
  return __builtin_amdgcn_mov_dpp(x, 0x120 + N, 0xF, 0xF, true);
}
__device__ __forceinline__ int min16(int x) {
  x = min(x, turned<1>(x));
  x = min(x, turned<2>(x));
  x = min(x, turned<4>(x));
  return __builtin_amdgcn_readfirstlane(min(x, turned<8>(x)));
}
__device__ __forceinline__ int max16(int x) {
  x = max(x, turned<1>(x));
  x = max(x, turned<2>(x));
  x = max(x, turned<4>(x));
  return __builtin_amdgcn_readfirstlane(max(x, turned<8>(x)));
}

// 32 positions' keys and values, lane (r16, q4): keys 16 g + r16, dimensions 32 k + 8 q4 ..; values of positions
// 512 / D i + lane / (D / 8), dimensions 8 (lane % (D / 8)) ..
template <class E, int D>
struct Rows {
  u32x4 k[2][D / 32], v[D / 16];
  int shown;  // a bit for each 16 positions: a page holds them
};

template <class E, int D, bool CAP, bool BIAS>
__global__ __launch_bounds__(64 * kWaves, D == 256 ? 1 : 2) void few_kernel(CoreArgs a, int tiles, int least) {
  typedef typename Vec<E>::x8 x8;
  constexpr bool BENT = CAP || BIAS;
  constexpr int KQ = D / 32, MT = D / 16, LR = 512 / D;  // LR rows of values a load
  constexpr int LD = D + 16;  // 8 banks further each row: the transposed reads of 8 rows meet no bank twice
  __shared__ __align__(16) E vt[kWaves][kHalf * LD];
  __shared__ float wm[kWaves][16], wl[kWaves][16];
  static_assert(kHalf * LD * sizeof(E) >= 16 * D * sizeof(float), "the waves' O^T pass through their value tiles");
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, q4 = lane >> 4;
  // The last slice of the launch is for the rows of padding behind the requests', "request N".
  const int s = blockIdx.z, splits = gridDim.z - 1, h = blockIdx.y;
  const bool padding = s == splits;
  if (padding && blockIdx.x >= kPadding) return;
  // the low bits of requests are turned with head and part, so that those meet all XCDs
  const int turn = (h + s) & (((int)gridDim.x & -(int)gridDim.x) - 1) & 7, bx = padding ? blockIdx.x : blockIdx.x ^ turn;
  const int r = padding ? a.N : tiles == 1 ? bx : bx / tiles;
  const int tile0 = padding ? bx : tiles == 1 ? 0 : bx - r * tiles;
  if (!padding && r >= a.N) return;
  if (padding) tiles = min((int)gridDim.x, kPadding);
  const int T = (int)a.T, group = a.group.d;
  const int from = r == 0 ? 0 : min(max(a.starts[r], 0), T);
  const int to = padding ? T : min(max(a.starts[r + 1], from), T);
  const int rows = (to - from) * group, size = 1 << a.page_shift;
  const int room = (int)min((int64_t)a.columns << a.page_shift, (int64_t)kAttendRoom);
  // the exponent's factor of the plain scores, never 0: a masked score stays -infinity
  const float c = BENT ? 1.f : fmaxf(fabsf(a.scale) * 1.44269504088896341f, 1.17549435e-38f);

  for (int tile = tile0; tile * 16 < rows; tile += tiles) {
    const int rho = tile * 16 + r16;
    const bool real = rho < rows;
    const int row_t = real ? a.group.of(rho) : 0;
    const int t = from + row_t, head = h * group + (real ? rho - row_t * group : 0);
    x8 qf[KQ];
    {
      const E* q = static_cast<const E*>(a.q) + t * a.q_token + head * a.q_head + 8 * q4;
#pragma unroll
      for (int k = 0; k < KQ; ++k) {
        u32x4 w = real ? *reinterpret_cast<const u32x4*>(q + 32 * k) : u32x4{0, 0, 0, 0};
        if (!BENT && a.scale < 0.f) w ^= 0x80008000u;
        qf[k] = __builtin_bit_cast(x8, w);
      }
    }
    const Bend bend(a.scale, CAP ? a.cap : 0.f, BIAS ? a.slopes : nullptr, head);
    // the block table's next 64 entries, an entry a lane, from position `at` on
    const auto entries = [&](int at) {
      const int column = (at >> a.page_shift) + lane;
      return column < a.columns ? a.tables[r * a.table_stride + column] : -1;
    };
    // without a window the part's first positions, and with them its pages, are known before the rows' limits
    const int early = a.window <= 0 && r < a.N ? entries((s * least + wave) * kStep) : -1;
    int lo, hi;
    attend_limits(real && r < a.N ? a.visible[t] : 0, a.window, room, lo, hi);
    const int stands = BIAS ? (real && r < a.N ? (a.positions ? a.positions[t] : a.visible[t] - 1) : 0) : 0;
    // over the rows that see anything: from the first position any of them sees to the last, and the
    // range that all of them see, where nothing is masked
    const int first = min16(hi > 0 ? lo : INT32_MAX), last = max16(hi);
    const int low = max16(lo), high = min16(real ? hi : INT32_MAX);
    const int begin = last > 0 ? first & ~(kStep - 1) : 0;
    const int steps = (last - begin + kStep - 1) / kStep;
    // with a window the rows' limits may lie further apart than the launch was made for: longer parts then
    const int per = max(least, ((steps + splits - 1) / splits + kWaves - 1) & ~(kWaves - 1));
    const int stop = min(steps, (s + 1) * per);
    if (padding ? splits > 1 : s > 0 && s * per >= steps) {  // nothing here: only the join hears of it
      if (tid < 16 && real)
        for (int part = padding ? 0 : s; part < (padding ? splits : s + 1); ++part) {
          float* ml = a.ws + a.T * a.heads * splits * D + (((int64_t)t * a.heads + head) * splits + part) * 2;
          ml[0] = -INFINITY;
          ml[1] = 0.f;
        }
      continue;
    }

    f32x4 o[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) o[i] = zero4();
    float m = hi > 0 ? -INFINITY : 0.f, l = 0.f;
    E* const vw = vt[wave];

    int i = s * per + wave;
    while (i < stop) {
      // 64 entries: the steps they serve find their pages without a load
      int pos = begin + i * kStep;
      const int column0 = pos >> a.page_shift;
      const int table = a.window <= 0 && i == s * per + wave ? early : entries(pos);
      const int64_t reach = (int64_t)(column0 + 64) << a.page_shift;  // the first position beyond them
      const int end = (int)min((int64_t)stop, (reach - begin) / kStep);
      // 32 positions on their way into registers; an entry that names no page reads as zeros
      const auto load = [&](Rows<E, D>& x, int at, bool any) {
        x.shown = 0;
        __amdgpu_buffer_rsrc_t page[2];
        int key[2];
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const uint32_t id = __builtin_amdgcn_readlane(table, (((at + 16 * g) >> a.page_shift) - column0) & 63);
          const bool ok = any && id < a.page_count;
          page[g] = buf_rsrc(a.data + ((uint64_t)(ok ? id : 0u) * a.kv_heads + h) * (uint64_t)(4 * size * D), ok ? 4 * size * D : 0);
          key[g] = ok ? ((at + 16 * g) & (size - 1)) * (2 * D) : 0;  // scalar: buf_rsrc's rule
          x.shown |= ok ? 1 << g : 0;
        }
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
          for (int k = 0; k < KQ; ++k) x.k[g][k] = buf_ld16<u32x4>(page[g], r16 * (2 * D) + 64 * k + 16 * q4, key[g]);
        __builtin_amdgcn_sched_barrier(0);  // keys before values, so that a wait for them is not one for both
#pragma unroll
        for (int n = 0; n < MT; ++n) {
          const int g = n / (MT / 2);
          const int value = x.shown >> g & 1 ? key[g] + 2 * size * D + n % (MT / 2) * (LR * 2 * D) : 0;
          x.v[n] = buf_ld16<u32x4>(page[g], 16 * lane, value);
        }
        __builtin_amdgcn_sched_barrier(0);
      };
      Rows<E, D> x;
      load(x, pos, true);
#pragma unroll 1
      for (; i < end; i += kWaves, pos += kWaves * kStep) {
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          const int at = pos + kHalf * half;
          f32x4 sc[2];
#pragma unroll
          for (int g = 0; g < 2; ++g) sc[g] = zero4();
#pragma unroll
          for (int k = 0; k < KQ; ++k)
#pragma unroll
            for (int g = 0; g < 2; ++g) sc[g] = mfma(__builtin_bit_cast(x8, x.k[g][k]), qf[k], sc[g]);
          if constexpr (BENT) {
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                sc[g][e] = CAP ? bend.capped(sc[g][e], bend.cap) : sc[g][e] * bend.c;
                if constexpr (BIAS)
                  sc[g][e] = __builtin_fmaf(-bend.slope, fabsf((float)__builtin_elementwise_sub_sat(stands, at + 16 * g + 4 * q4 + e)), sc[g][e]);
              }
          }
          // where not every row sees every position, hidden ones leave the scores, and values that are not finite reach
          // only the rows that see them
          bool odd = false;
          if (!(at >= low && at + kHalf <= high && x.shown == 3)) {
            const int lo0 = lo - at - 4 * q4, hi0 = hi - at - 4 * q4;
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if ((int)(16 * g + e < lo0) | (int)(16 * g + e >= hi0) | (int)!(x.shown >> g & 1)) sc[g][e] = -INFINITY;
            uint32_t any = 0;
#pragma unroll
            for (int n = 0; n < MT; ++n) any |= odd_values<E>(x.v[n]);
            odd = __any(any != 0);
          }
          x8 pf;
          float sum;
          const auto weights = [&] {
            const float base = kAttendBias<E> - (m == -INFINITY ? 0.f : m);
            sum = 0.f;
            f32x8 p;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e >> 2][e & 3], c, base));
              sum += p[e];
            }
            pf = to8<E>(p);
          };
          weights();
          // where the weights have grown too large, or are a row's first, its maximum moves and they are made again
          bool large = sum > kAttendLimit<E> || m == -INFINITY;
          if (__any(large)) {
            large = __shfl_xor((int)large, 16, 64) || large;  // the four lanes of a row
            large = __shfl_xor((int)large, 32, 64) || large;
            float top = sc[0][0];
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
              for (int e = 0; e < 4; ++e) top = fmaxf(top, sc[g][e]);
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64)) * c;
            if (large && top > m) {
              const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
              m = top;
              l *= f;
#pragma unroll
              for (int k = 0; k < MT; ++k) o[k] *= f;
            }
            weights();
          }
          l += sum;
          // the values through the wave's tile, which its LDS operations reach in order
          const auto put = [&](bool finite) {
#pragma unroll
            for (int n = 0; n < MT; ++n) {
              const x8 v = __builtin_bit_cast(x8, x.v[n]);
              st8(vw + (n * LR + lane / (D / 8)) * LD + 8 * (lane % (D / 8)), finite ? finite_values<E>(v) : v);
            }
          };
          put(odd);
#pragma unroll
          for (int k = 0; k < MT; ++k) o[k] = mfma(ld8_trpv<E>(vw, LD, 0, 16 * k), pf, o[k]);
          if (odd) {
            put(false);
#pragma unroll 1
            for (int j = 0; j < kHalf; ++j) {
              const bool seen = at + j >= lo && at + j < hi && (x.shown >> (j >> 4) & 1);
#pragma unroll
              for (int k = 0; k < MT; ++k) {
                const auto v = ld4(vw + j * LD + 16 * k + 4 * q4);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float f = (float)v[e];
                  if (seen && !(f - f == 0.f)) o[k][e] += f;
                }
              }
            }
          }
          // beyond the last step: of no page, which costs no memory traffic
          const bool more = half == 0 || i + kWaves < end;
          load(x, half == 0 ? at + kHalf : pos + kWaves * kStep, more);
        }
      }
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    // join the waves: O^T rows through LDS, their 16-byte columns XORed with the row against bank conflicts
    if (q4 == 0) {
      wm[wave][r16] = m;
      wl[wave][r16] = l;
    }
#pragma unroll
    for (int k = 0; k < MT; ++k)
      *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(vw) + r16 * D + 4 * ((4 * k + q4) ^ r16)) = o[k];
    __syncthreads();
    const int row = tid >> 4, n = tile * 16 + row, n_t = a.group.of(n);
    const int64_t at = (int64_t)(from + n_t) * a.heads + h * group + n - n_t * group;
    float M = wm[0][row], L = 0.f, f[kWaves];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) M = fmaxf(M, wm[w][row]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      f[w] = wm[w][row] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(wm[w][row] - M);
      L += f[w] * wl[w][row];
    }
    const int lo_n = __shfl(lo, row, 64), hi_n = __shfl(hi, row, 64);
    // no weight above 0: the row's positions are hidden here, or the scores of all are -infinity
    if (L == 0.f && hi_n > 0 && pages_hold(a, r, max(lo_n, begin + s * per * kStep), min(hi_n, begin + stop * kStep)))
      L = splits > 1 ? kNoWeight : __builtin_nanf("");
    if (n < rows) {
#pragma unroll
      for (int k = 0; k < D / 64; ++k) {
        const int col = (tid & 15) + 16 * k;
        f32x4 y = zero4();
#pragma unroll
        for (int w = 0; w < kWaves; ++w)
          y += f[w] * *reinterpret_cast<const f32x4*>(reinterpret_cast<float*>(vt[w]) + row * D + 4 * (col ^ row));
        if (splits == 1)
          st4(static_cast<E*>(a.out) + at * D + 4 * col, L == 0.f ? zero4() : y * (1.f / L));
        else if (L != 0.f)  // the join reads no part that saw nothing
          *reinterpret_cast<f32x4*>(a.ws + (at * splits + s) * D + 4 * col) = y;
      }
      if ((tid & 15) == 0) {
        if (splits > 1) {
          float* ml = a.ws + a.T * a.heads * splits * D + (at * splits + s) * 2;
          ml[0] = L == 0.f ? -INFINITY : M;
          ml[1] = L;
        } else if (a.lse) {
          a.lse[at] = (M - kAttendBias<E> + log2f(L)) * 0.693147180559945309f;
        }
      }
    }
    __syncthreads();
  }
}

template <class E, int D>
void launch_dim(const CoreArgs& a, int splits, int per, hipStream_t st) {
  const int group = a.heads / a.kv_heads;
  const int64_t each = (int64_t)(a.N + 1) * a.kv_heads * splits;
  const int tiles = (int)std::max<int64_t>(1, std::min<int64_t>(((int64_t)a.max_queries * group + 15) / 16, (1 << 23) / each));
  // a workgroup takes every tiles-th tile: none is left out whatever the bound
  const dim3 grid((unsigned)std::max<int64_t>(1, (int64_t)a.N * tiles), a.kv_heads, splits + 1);
  by_scores(a, [&](auto cap, auto bias) {
    few_kernel<E, D, decltype(cap)::value, decltype(bias)::value><<<grid, 64 * kWaves, 0, st>>>(a, tiles, per);
  });
}

template <class E>
void by_dim(const CoreArgs& a, int splits, int per, hipStream_t st) {
  if (a.D == 64)
    launch_dim<E, 64>(a, splits, per, st);
  else if (a.D == 128)
    launch_dim<E, 128>(a, splits, per, st);
  else
    launch_dim<E, 256>(a, splits, per, st);
}

}  // namespace

void launch_core_few(const CoreArgs& a, int splits, int per, hipStream_t st) {
  if (a.fp16)
    by_dim<f16>(a, splits, per, st);
  else
    by_dim<bf16>(a, splits, per, st);
}

}  // namespace cqgdn
