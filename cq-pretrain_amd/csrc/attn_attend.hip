// Attention of a step's query rows over the 4-bit pages.
//
// Row (t, query head) sees the positions [max(0, visible - window), visible) of its request and gets
// sum_j p_j v_j / sum_j p_j with p_j = exp(scale q k_j - m), in one pass over the positions with a
// running maximum m.  Rows of one request and one key head (new tokens x query heads of the group) are
// the columns of S^T = K Q^T, 16 at a time, so a lane owns one row: its limits, maximum and sum are the
// lane's own, and S^T's layout is already the operand of O^T = V^T P^T.
//
// Scores, sums and O are fp32.  The weights are rounded once to the rows' type, as the operand of that product, which
// moves a result by at most half a step of the type times sum_j p_j |v_j| / sum_j p_j, as much as rounding the result
// itself; sums of weights take them as they were.  Two terms of the type for a weight would double V's MFMAs.
//
// Few rows read each code once and are bound by that, or by latency.  64 ragged requests of up to 8192 positions (169
// MB): 37 us and 5 for the join, 4.6 TB/s; five of up to 65536, D = 256 (109 MB): 29 and 4; one of 9216: 8 and 4, of
// which the codes are one.  What it took: the parts' equal length (one eighth of the time), pages found without a load
// in the loop (each step waited for all that was under way), waits for keys apart from those for values, operands of V
// read from LDS three MFMAs early, and nothing spilled (the 11 KB a wave that were cost a third).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attn_kernels.hpp"
#include "attn_kv4.hpp"
#include "attn_plan.hpp"

namespace cqgdn {
namespace {

constexpr int kPadding = 16;  // workgroups a key head for rows behind the requests'

// The pages of a step's four 16 positions, the same for all lanes.  An entry that names no page reads as zeros (its
// buffer has no bytes, and takes no scalar offset: buf_rsrc's rule), and its positions are hidden.
struct Pages {
  const uint8_t* base[4];
  int shown;  // a bit each
  template <int D>
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t page(int g, int size) const {
    return buf_rsrc(base[g], shown >> g & 1 ? kv4_page_bytes(size, D) : 0);
  }
  // the scalar offset of a place in page g
  __device__ __forceinline__ int place(int g, int offset) const { return shown >> g & 1 ? offset : 0; }
};

// The codes of a step's keys and their scale bytes.  Lane (r16, q4) holds key r16 of each 16: 16 bytes from
// every 128 dimensions (8 where D is 64), which are one block of 32, so an MFMA step's K index (q4, j) stands
// for dimension 128 x + 32 q4 + 8 kk + j and Q is read likewise.
template <int D>
struct Keys {
  static constexpr int XK = D > 128 ? D / 128 : 1;  // loads of 16 keys
  static constexpr int WK = D >= 128 ? 4 : 2;       // words of one
  uint32_t w[4][XK][WK];
  uint8_t s[4][XK];
};
template <int D>
__device__ __forceinline__ void load_keys(Keys<D>& c, const Pages& p, int pos, int size, int lane) {
  const int r16 = lane & 15, q4 = lane >> 4;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int at = (pos + 16 * g) & (size - 1);
    const int codes = p.place(g, at * (D / 2)), scales = p.place(g, size * D + at * (D / 32));
    const __amdgpu_buffer_rsrc_t rs = p.template page<D>(g, size);
#pragma unroll
    for (int x = 0; x < Keys<D>::XK; ++x) {
      if constexpr (D >= 128) {
        const u32x4 w = buf_ld16<u32x4>(rs, r16 * (D / 2) + 16 * q4 + 64 * x, codes);
#pragma unroll
        for (int i = 0; i < 4; ++i) c.w[g][x][i] = w[i];
        c.s[g][x] = __builtin_amdgcn_raw_buffer_load_b8(rs, r16 * (D / 32) + q4 + 4 * x, scales, 0);
      } else {
        const auto w = __builtin_amdgcn_raw_buffer_load_b64(rs, r16 * (D / 2) + 8 * q4, codes, 0);
        c.w[g][x][0] = w[0];
        c.w[g][x][1] = w[1];
        c.s[g][x] = __builtin_amdgcn_raw_buffer_load_b8(rs, r16 * (D / 32) + (q4 >> 1), scales, 0);
      }
    }
  }
}

// Of the values, up to 128 dimensions of 32 positions at a time: PC lanes a position hold 32 of them each.
template <int D>
struct Values {
  static constexpr int DC = D < 128 ? D : 128, PC = DC / 32, J = DC / 64;
  u32x4 w[D / DC][2][J];
  uint8_t s[D / DC][2][J];
  static __device__ __forceinline__ int position(int half, int j, int lane) { return 32 * half + 64 / PC * j + lane / PC; }
};
template <int D>
__device__ __forceinline__ void load_values(Values<D>& c, const Pages& p, int pos, int size, int lane) {
  typedef Values<D> V;
#pragma unroll
  for (int half = 0; half < 2; ++half)
#pragma unroll
    for (int j = 0; j < V::J; ++j) {
      const int g = 2 * half + j, at = (pos + 16 * g) & (size - 1);
      const int codes = p.place(g, size * (D / 2) + at * (D / 2));
      const int scales = p.place(g, size * D + size * (D / 32) + at * (D / 32));
#pragma unroll
      for (int x = 0; x < D / V::DC; ++x) {
        if constexpr (D >= 128) {
          c.w[x][half][j] = buf_ld16<u32x4>(p.template page<D>(g, size), lane / 4 * (D / 2) + lane % 4 * 16 + 64 * x, codes);
          c.s[x][half][j] = __builtin_amdgcn_raw_buffer_load_b8(p.template page<D>(g, size), lane / 4 * (D / 32) + lane % 4 + 4 * x, scales, 0);
        } else {
          // 32 positions a load, which two pages may hold: a lane's offset lies beyond the one that is not its own
          const int at1 = (pos + 16 * g + 16) & (size - 1), none = 1 << 30;
          const int codes1 = p.place(g + 1, size * (D / 2) + at1 * (D / 2));
          const int scales1 = p.place(g + 1, size * D + size * (D / 32) + at1 * (D / 32));
          const int lo = lane < 32 ? lane * 16 : none, hi = lane < 32 ? none : (lane - 32) * 16;
          const int slo = lane < 32 ? lane : none, shi = lane < 32 ? none : lane - 32;
          c.w[x][half][j] = buf_ld16<u32x4>(p.template page<D>(g, size), lo, codes) |
                            buf_ld16<u32x4>(p.template page<D>(g + 1, size), hi, codes1);
          c.s[x][half][j] = __builtin_amdgcn_raw_buffer_load_b8(p.template page<D>(g, size), slo, scales, 0) |
                            __builtin_amdgcn_raw_buffer_load_b8(p.template page<D>(g + 1, size), shi, scales1, 0);
        }
      }
    }
}

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

// One workgroup: 16 rows of one request and key head, one of `splits` parts of the positions, `least` steps
// long (the last parts, which are empty where requests are shorter, come last).  The waves' steps interleave,
// each with its own maximum, sum and O^T, and are joined at the end.  A step's codes are on their way from the
// moment those before have been used, in registers.
template <class E, int D>
__global__ __launch_bounds__(64 * kWaves, D == 256 ? 2 : 3) void attend_kernel(AttendArgs a, int tiles, int least) {
  typedef typename Vec<E>::x8 x8;
  typedef Values<D> V;
  constexpr int DC = V::DC, LD = DC + 16;  // 8 banks further each row: the transposed reads of 8 rows meet no bank twice
  constexpr int KQ = D / 32, MT = D / 16;
  __shared__ __align__(16) E vt[kWaves][32 * LD];
  __shared__ float wm[kWaves][16], wl[kWaves][16];
  static_assert(32 * LD * sizeof(E) >= 16 * DC * sizeof(float), "the waves' O^T pass through their value tiles");
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, q4 = lane >> 4;
  // The last slice of the launch is for the rows of padding behind the requests', "request N".  Were its workgroups
  // between the others, those would meet every second XCD only where there is one request
  // (of 9216 positions: 12.2 us against 11.2).
  const int s = blockIdx.z, splits = gridDim.z - 1, h = blockIdx.y;
  const bool padding = s == splits;
  if (padding && blockIdx.x >= kPadding) return;
  // Workgroups go to the XCDs in turn: where the requests are a multiple of some power of two, each would meet the
  // same XCDs with all its heads and parts, the longest too.  Their low bits are turned within that power (64 ragged
  // requests: 48.1 us without, 45.8 with).
  const int turn = (h + s) & (((int)gridDim.x & -(int)gridDim.x) - 1) & 7, x = padding ? blockIdx.x : blockIdx.x ^ turn;
  const int r = padding ? a.N : tiles == 1 ? x : x / tiles;
  const int tile0 = padding ? x : tiles == 1 ? 0 : x - r * tiles;
  if (!padding && r >= a.N) return;
  if (padding) tiles = min((int)gridDim.x, kPadding);
  const int T = (int)a.T, group = a.group.d;
  const int from = r == 0 ? 0 : min(max(a.starts[r], 0), T);
  const int to = padding ? T : min(max(a.starts[r + 1], from), T);
  const int rows = (to - from) * group, size = 1 << a.page_shift;
  const int room = (int)min((int64_t)a.columns << a.page_shift, (int64_t)kAttendRoom);
  const uint8_t* const head_base = a.data + (int64_t)h * kv4_page_bytes(size, D);
  const uint64_t stride = (uint64_t)a.kv_heads * kv4_page_bytes(size, D);
  // the exponent's factor, never 0: a masked score stays -infinity; its sign goes with Q
  const float c = fmaxf(fabsf(a.scale) * 1.44269504088896341f, 1.17549435e-38f);

  for (int tile = tile0; tile * 16 < rows; tile += tiles) {
    const int rho = tile * 16 + r16;
    const bool real = rho < rows;
    const int row_t = real ? a.group.of(rho) : 0;
    const int t = from + row_t, head = h * group + (real ? rho - row_t * group : 0);
    x8 qf[KQ];
    {
      const E* q = static_cast<const E*>(a.q) + t * a.q_token + head * a.q_head;
#pragma unroll
      for (int k = 0; k < KQ; ++k) {
        u32x4 w = real ? *reinterpret_cast<const u32x4*>(q + (D >= 128 ? 128 * (k / 4) + 32 * q4 + 8 * (k % 4) : 16 * q4 + 8 * k))
                       : u32x4{0, 0, 0, 0};
        if (a.scale < 0.f) w ^= 0x80008000u;
        qf[k] = __builtin_bit_cast(x8, w);
      }
    }
    // the block table's next 64 entries, an entry a lane, from position `at` on
    const auto entries = [&](int at) {
      const int column = (at >> a.page_shift) + lane;
      return column < a.columns ? a.tables[r * a.table_stride + column] : -1;
    };
    // without a window the part's first positions, and with them its pages, are known before the rows' limits
    const int early = a.window <= 0 && r < a.N ? entries((s * least + wave) * kStep) : -1;
    int lo, hi;
    attend_limits(real && r < a.N ? a.visible[t] : 0, a.window, room, lo, hi);
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
    uint32_t nan = 0;  // blocks of 32 dimensions in which the row sees a NaN value
    E* const vw = vt[wave];

    int i = s * per + wave;
    while (i < stop) {
      // 64 entries: the steps they serve find their pages without a load
      int pos = begin + i * kStep;
      const int column0 = pos >> a.page_shift;
      const int table = a.window <= 0 && i == s * per + wave ? early : entries(pos);
      const int64_t reach = (int64_t)(column0 + 64) << a.page_shift;  // the first position beyond them
      const int end = (int)min((int64_t)stop, (reach - begin) / kStep);
      const auto find = [&](int at, bool any) {
        Pages x;
        x.shown = 0;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const uint32_t page = __builtin_amdgcn_readlane(table, (((at + 16 * g) >> a.page_shift) - column0) & 63);
          const bool ok = any && page < a.page_count;
          x.base[g] = head_base + (ok ? page : 0u) * stride;
          x.shown |= ok ? 1 << g : 0;
        }
        return x;
      };
      Keys<D> keys;
      V values;
      int shown;
      {
        const Pages p = find(pos, true);
        load_keys<D>(keys, p, pos, size, lane);
        __builtin_amdgcn_sched_barrier(0);  // keys before values, so that a wait for them is not one for both
        load_values<D>(values, p, pos, size, lane);
        __builtin_amdgcn_sched_barrier(0);
        shown = p.shown;
      }
#pragma unroll 1
      for (; i < end; i += kWaves, pos += kWaves * kStep) {
        f32x4 sc[4];
        float ks[4][Keys<D>::XK];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          sc[g] = zero4();
#pragma unroll
          for (int x = 0; x < Keys<D>::XK; ++x) ks[g][x] = kv4_scale(keys.s[g][x]);
        }
#pragma unroll
        for (int x = 0; x < Keys<D>::XK; ++x)
#pragma unroll
          for (int w = 0; w < Keys<D>::WK; ++w)
#pragma unroll
            for (int g = 0; g < 4; ++g)
              sc[g] = mfma(kv4_values<E>(keys.w[g][x][w], ks[g][x]), qf[x * Keys<D>::WK + w], sc[g]);
        // beyond the last step: of no page, which costs no memory traffic
        const Pages next = find(pos + kWaves * kStep, i + kWaves < end);
        load_keys<D>(keys, next, pos + kWaves * kStep, size, lane);
        __builtin_amdgcn_sched_barrier(0);
        // where not every row sees every position, hidden ones leave the scores, a position that none sees is
        // zero among the values, and a NaN reaches only the rows that see it
        if (!(pos >= low && pos + kStep <= high && shown == 15)) {
          const int lo0 = lo - pos, hi0 = hi - pos;
#pragma unroll
          for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int at = 16 * g + e;  // and 4 q4
              if ((int)(at < lo0 - 4 * q4) | (int)(at >= hi0 - 4 * q4) | (int)!(shown >> g & 1)) sc[g][e] = -INFINITY;
            }
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int x = 0; x < D / DC; ++x)
#pragma unroll
              for (int j = 0; j < V::J; ++j) {
                const int tok = V::position(half, j, lane);
                const bool any = pos + tok >= first && pos + tok < last, is_nan = values.s[x][half][j] == 255;
                for (uint64_t bad = __ballot(any && is_nan); bad; bad &= bad - 1) {
                  const int n = __builtin_ctzll(bad), at = V::position(half, j, n);
                  nan |= at >= lo0 && at < hi0 ? 1u << (V::PC * x + n % V::PC) : 0u;
                }
                if (!any || is_nan) {
                  values.w[x][half][j] = u32x4{0, 0, 0, 0};
                  values.s[x][half][j] = 0;
                }
              }
        }
        x8 pf[2];
        float sum;
        const auto weights = [&] {
          const float base = kAttendBias<E> - (m == -INFINITY ? 0.f : m);
          sum = 0.f;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            f32x8 p;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[2 * half + (e >> 2)][e & 3], c, base));
              sum += p[e];
            }
            pf[half] = to8<E>(p);
          }
        };
        weights();
        // where the weights have grown too large, or are a row's first, its maximum moves and they are made again
        bool large = sum > kAttendLimit<E> || m == -INFINITY;
        if (__any(large)) {
          large = __shfl_xor((int)large, 16, 64) || large;  // the four lanes of a row
          large = __shfl_xor((int)large, 32, 64) || large;
          float top = sc[0][0];
#pragma unroll
          for (int g = 0; g < 4; ++g)
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
        // values: chunk (half, x) passes through the wave's tile, whose operands are read kEarly MFMAs ahead of
        // their own (a wave's LDS operations complete in order)
        constexpr int OPS = DC / 16, ALL = 2 * (D / DC) * OPS, kEarly = 3;
        x8 vf[ALL];
        const auto ahead = [&](int i) {
          const int chunk = i / OPS, half = chunk / (D / DC), x = chunk % (D / DC);
          if (i % OPS == 0) {
#pragma unroll
            for (int j = 0; j < V::J; ++j) {
              const int tok = V::position(half, j, lane), piece = lane % V::PC;
              const float vs = kv4_scale(values.s[x][half][j]);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                st8(vw + (tok - 32 * half) * LD + 32 * piece + 8 * e, kv4_values<E>(values.w[x][half][j][e], vs));
            }
          }
          vf[i] = ld8_trpv<E>(vw, LD, 0, i % OPS * 16);
        };
#pragma unroll
        for (int i = 0; i < kEarly; ++i) ahead(i);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < ALL; ++i) {
          if (i + kEarly < ALL) ahead(i + kEarly);
          const int chunk = i / OPS, at = chunk % (D / DC) * OPS + i % OPS;
          o[at] = mfma(vf[i], pf[chunk / (D / DC)], o[at]);
          __builtin_amdgcn_sched_barrier(0);
        }
        load_values<D>(values, next, pos + kWaves * kStep, size, lane);
        shown = next.shown;
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (__any(nan != 0)) {
#pragma unroll
      for (int k = 0; k < MT; ++k)
        if (nan >> (k / 2) & 1) o[k] = zero4() + __builtin_nanf("");
    }
    // join the waves: O^T rows through LDS, DC dimensions at a time, their 16-byte columns XORed with the row
    // against bank conflicts
    int late = tid;  // what follows is worked out here, not held in registers through the loop
    asm volatile("" : "+v"(late));
    const int lr = late & 15, lq = late >> 4 & 3;
    if (lq == 0) {
      wm[wave][lr] = m;
      wl[wave][lr] = l;
    }
    const int row = late >> 4, n = tile * 16 + row, n_t = a.group.of(n);
    const int64_t at = (int64_t)(from + n_t) * a.heads + h * group + n - n_t * group;
    float M, L = 0.f, f[kWaves];
#pragma unroll
    for (int x = 0; x < D / DC; ++x) {
#pragma unroll
      for (int k = 0; k < DC / 16; ++k)
        *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(vw) + lr * DC + 4 * ((4 * k + lq) ^ lr)) = o[DC / 16 * x + k];
      __syncthreads();
      if (x == 0) {
        M = wm[0][row];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) M = fmaxf(M, wm[w][row]);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          f[w] = wm[w][row] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(wm[w][row] - M);
          L += f[w] * wl[w][row];
        }
      }
      if (n < rows) {
#pragma unroll
        for (int k = 0; k < DC / 64; ++k) {
          const int col = (late & 15) + 16 * k;
          f32x4 y = zero4();
#pragma unroll
          for (int w = 0; w < kWaves; ++w)
            y += f[w] * *reinterpret_cast<const f32x4*>(reinterpret_cast<float*>(vt[w]) + row * DC + 4 * (col ^ row));
          if (splits == 1)
            st4(static_cast<E*>(a.out) + at * D + DC * x + 4 * col, L == 0.f ? zero4() : y * (1.f / L));
          else if (L != 0.f)  // the join reads no part that saw nothing
            *reinterpret_cast<f32x4*>(a.ws + (at * splits + s) * D + DC * x + 4 * col) = y;
        }
      }
      __syncthreads();
    }
    if (n < rows && (late & 15) == 0) {
      if (splits > 1) {
        float* ml = a.ws + a.T * a.heads * splits * D + (at * splits + s) * 2;
        ml[0] = L == 0.f ? -INFINITY : M;
        ml[1] = L;
      } else if (a.lse) {
        a.lse[at] = (M - kAttendBias<E> + log2f(L)) * 0.693147180559945309f;
      }
    }
  }
}

// Joins the parts of many rows: D / 4 lanes a row, each taking its 4 dimensions through the parts.
template <class E, int D>
__global__ __launch_bounds__(256) void join_rows_kernel(AttendArgs a, int splits) {
  constexpr int L4 = D / 4, UP = 4;  // lanes a row, parts whose loads are under way at once
  const int64_t at = (int64_t)blockIdx.x * (256 / L4) + threadIdx.x / L4;
  const int col = threadIdx.x % L4;
  if (at >= a.T * a.heads) return;
  const float2* ml = reinterpret_cast<const float2*>(a.ws + a.T * a.heads * splits * D) + at * splits;
  const float* rows = a.ws + at * splits * D + 4 * col;
  float M = -INFINITY;
#pragma unroll 8
  for (int s = 0; s < splits; ++s) M = fmaxf(M, ml[s].x);
  f32x4 y = zero4();
  float L = 0.f;
  for (int s0 = 0; s0 < splits; s0 += UP) {
    f32x4 x[UP];
    float2 part[UP];
#pragma unroll
    for (int i = 0; i < UP; ++i) {
      const int s = min(s0 + i, splits - 1);
      part[i] = ml[s];
      x[i] = *reinterpret_cast<const f32x4*>(rows + s * D);
    }
#pragma unroll
    for (int i = 0; i < UP; ++i) {
      // a part that saw nothing wrote no row
      const bool none = s0 + i >= splits || (part[i].x == -INFINITY && part[i].y == 0.f);
      const float f = none ? 0.f : __builtin_amdgcn_exp2f(part[i].x - M);
      L += f * part[i].y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] += none ? 0.f : f * x[i][e];
    }
  }
  st4(static_cast<E*>(a.out) + at * D + 4 * col, L == 0.f ? zero4() : y * (1.f / L));
  if (a.lse && col == 0) a.lse[at] = (M - kAttendBias<E> + log2f(L)) * 0.693147180559945309f;
}

// Joins the parts of few rows, a workgroup for 64 dimensions of one: the parts' weights, then 16 parts at a time.
template <class E, int D>
__global__ __launch_bounds__(256) void join_kernel(AttendArgs a, int splits) {
  constexpr int W = kMaxSplits / 256;
  __shared__ float weight[kMaxSplits];
  __shared__ float red[2][4];
  __shared__ int count[4];
  __shared__ __align__(16) float part[16][64];
  const int64_t at = blockIdx.x / (D / 64);
  const int d0 = blockIdx.x % (D / 64) * 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = tid & 15, g = tid >> 4;
  const float2* ml = reinterpret_cast<const float2*>(a.ws + a.T * a.heads * splits * D) + at * splits;
  float2 mine[W];
  float M = -INFINITY, L = 0.f;
  int n = 0;  // parts up to the last that saw anything; the others wrote no row
#pragma unroll
  for (int j = 0; j < W; ++j) {
    const int s = tid + 256 * j;
    mine[j] = s < splits ? ml[s] : float2{-INFINITY, 0.f};
    M = fmaxf(M, mine[j].x);
    if (mine[j].x != -INFINITY || mine[j].y != 0.f) n = s + 1;
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    M = fmaxf(M, __shfl_xor(M, o, 64));
    n = max(n, __shfl_xor(n, o, 64));
  }
  if (lane == 0) {
    red[0][wave] = M;
    count[wave] = n;
  }
  __syncthreads();
  M = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  n = max(max(count[0], count[1]), max(count[2], count[3]));
#pragma unroll
  for (int j = 0; j < W; ++j) {
    const bool empty = mine[j].x == -INFINITY && mine[j].y == 0.f;
    const float f = empty ? 0.f : __builtin_amdgcn_exp2f(mine[j].x - M);
    weight[tid + 256 * j] = empty ? -1.f : f;
    L += f * mine[j].y;
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) L += __shfl_xor(L, o, 64);
  if (lane == 0) red[1][wave] = L;
  __syncthreads();
  L = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
  f32x4 y = zero4();
  const float* rows = a.ws + at * splits * D + d0 + 4 * col;
#pragma unroll 4
  for (int s = g; s < n; s += 16) {
    const f32x4 x = *reinterpret_cast<const f32x4*>(rows + s * D);
    const float f = weight[s];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] += f < 0.f ? 0.f : f * x[e];
  }
  *reinterpret_cast<f32x4*>(&part[g][4 * col]) = y;
  __syncthreads();
  if (tid < 16) {
#pragma unroll
    for (int k = 1; k < 16; ++k) y += *reinterpret_cast<const f32x4*>(&part[k][4 * col]);
    st4(static_cast<E*>(a.out) + at * D + d0 + 4 * col, L == 0.f ? zero4() : y * (1.f / L));
  }
  if (a.lse && tid == 0 && d0 == 0) a.lse[at] = (M - kAttendBias<E> + log2f(L)) * 0.693147180559945309f;
}

template <class E, int D>
void launch_dim(const AttendArgs& a, hipStream_t st) {
  const int group = a.heads / a.kv_heads;
  const AttendPlan p = attend_plan(a.N, a.kv_heads, group, D, a.max_queries, (int64_t)a.columns << a.page_shift, a.window);
  if (p.tiles) {
    launch_attend_tiles(a, p.splits, st);
  } else {
    const int64_t each = (int64_t)(a.N + 1) * a.kv_heads * p.splits;
    const int tiles = (int)std::max<int64_t>(1, std::min<int64_t>(((int64_t)a.max_queries * group + 15) / 16, (1 << 23) / each));
    // a workgroup takes every tiles-th tile: none is left out whatever the bound
    const dim3 grid((unsigned)std::max<int64_t>(1, (int64_t)a.N * tiles), a.kv_heads, p.splits + 1);
    attend_kernel<E, D><<<grid, 64 * kWaves, 0, st>>>(a, tiles, p.per);
  }
  if (p.splits > 1) {
    // 2048 rows of 33 MB in two parts: 60 us by the kernel for few rows; 32 rows in 36 parts: 4 us by it
    const int64_t groups = (a.T * a.heads * D + 1023) / 1024;
    if (groups >= 256)
      join_rows_kernel<E, D><<<(unsigned)groups, 256, 0, st>>>(a, p.splits);
    else
      join_kernel<E, D><<<(unsigned)(a.T * a.heads * (D / 64)), 256, 0, st>>>(a, p.splits);
  }
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
  const int splits = attend_plan(N, kv_heads, heads / kv_heads, D, max_queries, capacity, 0).splits;
  return splits > 1 ? (size_t)T * heads * splits * (D + 2) * sizeof(float) : 0;
}

void launch_attend(const AttendArgs& a, hipStream_t st) {
  if (a.fp16)
    by_dim<f16>(a, st);
  else
    by_dim<bf16>(a, st);
}

}  // namespace cqgdn
