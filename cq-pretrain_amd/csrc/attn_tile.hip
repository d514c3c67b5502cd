// Attention of many query rows a request over the 4-bit pages: a prompt's rows share the values of a page.
//
// The mathematics is that of attn_attend.hip.  Here a workgroup takes 128 rows of one request and key head,
// 32 a wave, and kTokens positions a step.  Its threads convert the step's codes once into K and V tiles of E in
// shared memory, two deep, so that the next step's codes are on their way and being converted while the
// waves multiply.  S^T = K Q^T and O^T = V^T P^T run on 32 x 32 x 16 MFMAs with a row a column, so a lane
// (and its partner 32 lanes on) owns a row: limits, maximum and sum stay in its registers, and S^T's layout
// is already an operand of O^T.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attn_kernels.hpp"
#include "attn_kv4.hpp"

namespace cqgdn {
namespace {

constexpr int kRows = 128;    // of a workgroup, 32 a wave

typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// Positions a step: 256 threads convert 32 values of K and of V each.
template <int D>
constexpr int kTokens = 8192 / D;

// K rows are 16 bytes longer than their values: read 16 bytes a lane, 16 rows at a time, they meet all 64 banks
// once.  V is read by quads of rows and 64 bytes of each; its 16-byte column c lies at v_column(row, c), the
// same for rows 4 apart, so that those meet all banks once as well.  Both are written 16 bytes a lane, every
// fourth column, again without a bank met twice.
template <int D>
constexpr int kStrideK = D + 8;
template <int D>
__device__ __forceinline__ int v_column(int row, int c) {
  if constexpr (D == 64) return c ^ (4 * ((row >> 1) & 1)) ^ ((row >> 1) & 3);
  return c ^ (5 * (row & 3)) ^ (D == 256 ? (c >> 4) << 1 : 0);
}

// what a thread fetches of a step: 32 values of K and of V
struct Piece {
  u32x4 k, v;
  uint32_t ks, vs;
  bool ok;
};

template <int D>
__device__ __forceinline__ Piece fetch(const AttendArgs& a, int page, int pos, int h, int piece) {
  Piece x;
  const int size = 1 << a.page_shift, at = pos & (size - 1);
  x.ok = page >= 0 && page < (int)a.page_count;  // an entry that names no page: its positions are hidden
  const uint8_t* base = a.data + ((int64_t)(x.ok ? page : 0) * a.kv_heads + h) * kv4_page_bytes(size, D);
  const uint8_t* code = base + at * (D / 2) + 16 * piece;
  const uint8_t* scale = base + size * D + at * (D / 32) + piece;
  x.k = *reinterpret_cast<const u32x4*>(code);
  x.v = *reinterpret_cast<const u32x4*>(code + size * (D / 2));
  x.ks = scale[0];
  x.vs = scale[size * (D / 32)];
  return x;
}

template <class E, int D>
__global__ __launch_bounds__(256, 2) void tile_kernel(AttendArgs a, int tiles, int splits) {
  typedef typename Vec<E>::x8 x8;
  constexpr int TOK = kTokens<D>, PV = D / 32, NS = TOK / 32, KQ = D / 16, MT = D / 32;
  __shared__ __align__(16) E kt[2][TOK * kStrideK<D>];
  __shared__ __align__(16) E vt[2][TOK * D];
  // of the positions each wave fetched: a bit for every 16 that are hidden, the sign for a NaN among the values
  __shared__ __align__(16) int marks[2][4];
  __shared__ uint64_t bad[2][4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n32 = lane & 31, kg = lane >> 5;
  // Launch order: a request's last tiles, which see most, first; every other round of 256 workgroups (one a
  // CU) reversed, so that a CU's workgroups add up to the same
  const int each = a.kv_heads * (a.N + 1) * splits;
  int b = blockIdx.x;
  if ((b >> 8 & 1) && (b | 255) < (int)gridDim.x) b ^= 255;
  const int tile0 = tiles - 1 - b / each;
  b %= each;
  const int s = b % splits;
  b /= splits;
  const int h = b % a.kv_heads, r = b / a.kv_heads;
  const int group = a.heads / a.kv_heads, T = (int)a.T;
  const int from = r == 0 ? 0 : min(max(a.starts[r], 0), T);
  const int to = r == a.N ? T : min(max(a.starts[r + 1], from), T);  // request N: the padding behind the last
  const int rows = (to - from) * group;
  const int room = (int)min((int64_t)a.columns << a.page_shift, (int64_t)INT32_MAX - 1024);
  const int token = tid / PV, piece = tid % PV;  // the thread's part of a step
  // the exponent's factor, never 0: a masked score stays -infinity; its sign goes with Q
  const float c = fmaxf(fabsf(a.scale) * 1.44269504088896341f, 1.17549435e-38f);
  constexpr float bias = kAttendBias<E>;
  typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
  // the lane's K row of a step, and its piece of V: tokens 4 kg + {0..3, 8..11} at dimension 32 k + n32 come
  // transposed out of quads of lanes
  const E* const kl = kt[0] + n32 * kStrideK<D> + 8 * kg;
  const E* vl[MT];
#pragma unroll
  for (int k = 0; k < MT; ++k) {
    const int j = lane & 15, row = 4 * kg + (j >> 2), col = 4 * k + 2 * (lane >> 4 & 1) + (j >> 1 & 1);
    vl[k] = vt[0] + row * D + 8 * v_column<D>(row, col) + 4 * (j & 1);
  }

  for (int tile = tile0; tile * kRows < rows; tile += tiles) {
    const auto limits = [&](int rho, int& lo, int& hi) {
      hi = rho < rows && r < a.N ? min(max(a.visible[from + rho / group], 0), room) : 0;
      lo = a.window > 0 ? max(0, hi - a.window) : 0;
    };
    // what the workgroup's rows see together
    int first, last;
    {
      int lo0, hi0, lo1, hi1;
      limits(tile * kRows + lane, lo0, hi0);
      limits(tile * kRows + 64 + lane, lo1, hi1);
      first = min(hi0 > 0 ? lo0 : INT32_MAX, hi1 > 0 ? lo1 : INT32_MAX);
      last = max(hi0, hi1);
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        first = min(first, __shfl_xor(first, o, 64));
        last = max(last, __shfl_xor(last, o, 64));
      }
      first = __builtin_amdgcn_readfirstlane(first);
      last = __builtin_amdgcn_readfirstlane(last);
    }
    const int rho = tile * kRows + 32 * wave + n32;
    const bool real = rho < rows;
    int lo, hi;
    limits(rho, lo, hi);
    // the wave's: the range that any of its rows sees, and the one all of them see, where nothing is masked
    int wfirst = hi > 0 ? lo : INT32_MAX, wlast = hi, low = lo, high = real ? hi : INT32_MAX;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      wfirst = min(wfirst, __shfl_xor(wfirst, o, 64));
      wlast = max(wlast, __shfl_xor(wlast, o, 64));
      low = max(low, __shfl_xor(low, o, 64));
      high = min(high, __shfl_xor(high, o, 64));
    }
    wfirst = __builtin_amdgcn_readfirstlane(wfirst);
    wlast = __builtin_amdgcn_readfirstlane(wlast);
    low = __builtin_amdgcn_readfirstlane(low);
    high = __builtin_amdgcn_readfirstlane(high);

    const int t = from + (real ? rho / group : 0), head = h * group + (real ? rho % group : 0);
    x8 qf[KQ];  // lane (n32, kg): row n32, dimensions 16 i + 8 kg ..
    {
      const E* q = static_cast<const E*>(a.q) + t * a.q_token + head * a.q_head + 8 * kg;
#pragma unroll
      for (int i = 0; i < KQ; ++i) {
        u32x4 w = real ? *reinterpret_cast<const u32x4*>(q + 16 * i) : u32x4{0, 0, 0, 0};
        if (a.scale < 0.f) w ^= 0x80008000u;
        qf[i] = __builtin_bit_cast(x8, w);
      }
    }
    f32x16 o[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) o[i] = f32x16{};
    float m = -INFINITY, l = 0.f;

    const int begin = last > 0 ? first & ~(TOK - 1) : 0;
    const int steps = (last - begin + TOK - 1) / TOK, per = (steps + splits - 1) / splits;
    const int stop = min(steps, (s + 1) * per);

    const auto store = [&](const Piece& x, int buf, int pos) {
      const int at = pos + token;
      // a position that no row sees is zero, and so is a NaN value: it goes to the rows that see it below
      const bool any = x.ok && at >= first && at < last, nan = any && x.vs == 255;
      const uint64_t hidden = __ballot(!x.ok), nans = __ballot(nan);
      if (lane == 0) {
        bad[buf][wave] = nans;
        marks[buf][wave] = (int)(hidden & 1) | (PV == 2 ? (int)(hidden >> 32 & 1) << 1 : 0) | (nans ? INT32_MIN : 0);
      }
      const float ks = kv4_scale(x.ks), vs = any && !nan ? kv4_scale(x.vs) : 0.f;
      const u32x4 v = any && !nan ? x.v : u32x4{0, 0, 0, 0};
      E* const kr = kt[buf] + token * kStrideK<D> + 32 * piece;
      E* const vr = vt[buf] + token * D;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        st8(kr + 8 * e, kv4_values<E>(x.k[e], ks));
        st8(vr + 8 * v_column<D>(token, 4 * piece + e), kv4_values<E>(v[e], vs));
      }
    };

    int i = s * per;
    if (i < stop) {
      Piece next = fetch<D>(a, page_of(a, r, begin + i * TOK + token), begin + i * TOK + token, h, piece);
      int pg = page_of(a, r, begin + (i + 1) * TOK + token);
      store(next, i & 1, begin + i * TOK);
      if (i + 1 < stop) next = fetch<D>(a, pg, begin + (i + 1) * TOK + token, h, piece);
      pg = page_of(a, r, begin + (i + 2) * TOK + token);
      __syncthreads();
      for (; i < stop; ++i) {
        const int pos = begin + i * TOK, buf = i & 1;
        if (i + 1 < stop) {
          store(next, buf ^ 1, pos + TOK);
          if (i + 2 < stop) next = fetch<D>(a, pg, pos + 2 * TOK + token, h, piece);
          pg = page_of(a, r, pos + 3 * TOK + token);
        }
        if (pos < wlast && pos + TOK > wfirst) {
          int mark[4];
#pragma unroll
          for (int w = 0; w < 4; ++w) mark[w] = __builtin_amdgcn_readfirstlane(marks[buf][w]);
          const bool clean = (mark[0] | mark[1] | mark[2] | mark[3]) == 0;
          f32x16 sc[NS];
#pragma unroll
          for (int u = 0; u < NS; ++u) {
            sc[u] = f32x16{};
#pragma unroll
            for (int k = 0; k < KQ; ++k)
              sc[u] = mfma32(ld8(kl + buf * (TOK * kStrideK<D>) + 32 * u * kStrideK<D> + 16 * k), qf[k], sc[u]);
          }
          if (!(clean && pos >= low && pos + TOK <= high)) {
            const int at0 = pos + 4 * kg;
#pragma unroll
            for (int u = 0; u < NS; ++u)
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                const int at = 32 * u + 8 * (e >> 2) + (e & 3), g = 2 * u + (e >> 3);
                const int word = D == 256 ? 2 * g : D == 128 ? g : g >> 1;
                const bool shown = !(mark[word] >> (D == 64 ? g & 1 : 0) & 1);
                if (at < lo - at0 || at >= hi - at0 || !shown) sc[u][e] = -INFINITY;
              }
          }
          float top = sc[0][0];
#pragma unroll
          for (int u = 0; u < NS; ++u)
#pragma unroll
            for (int e = 0; e < 16; ++e) top = fmaxf(top, sc[u][e]);
          top *= c;
          if (__any(top > m + kLazy)) {  // the maximum moves rarely, and for each row by itself
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            if (top > m + kLazy) {
              const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
              m = top;
              l *= f;
#pragma unroll
              for (int k = 0; k < MT; ++k) o[k] *= f;
            }
          }
          const float base = (m == -INFINITY ? 0.f : m) - bias;
          x8 pf[2 * NS];
#pragma unroll
          for (int u = 0; u < NS; ++u)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              f32x8 p;
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[u][8 * e + j], c, -base));
                l += p[j];
              }
              pf[2 * u + e] = to8<E>(p);
            }
          if (!clean) {  // NaN values: to the rows that see them, in their 32 dimensions
#pragma unroll 1
            for (int w = 0; w < 4; ++w)
#pragma unroll 1
              for (uint64_t x = bad[buf][w]; x; x &= x - 1) {
                const int n = 64 * w + __builtin_ctzll(x), at = pos + n / PV;
                const float add = at >= lo && at < hi ? __builtin_nanf("") : 0.f;
#pragma unroll
                for (int k = 0; k < MT; ++k)
                  if (k == n % PV) o[k] += add;
              }
          }
#pragma unroll
          for (int k = 0; k < MT; ++k)
#pragma unroll
            for (int u = 0; u < 2 * NS; ++u) {
              const E* p = vl[k] + buf * (TOK * D) + 16 * u * D;
              const i16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)p);
              const i16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(p + 8 * D));
              o[k] = mfma32(__builtin_bit_cast(x8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7)), pf[u], o[k]);
            }
        }
        __syncthreads();
      }
    }
    l += __shfl_xor(l, 32, 64);
    if (real) {
      const int64_t at = (int64_t)t * a.heads + head;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      if (splits == 1 || m != -INFINITY || l != 0.f) {  // the join reads no part that saw nothing
#pragma unroll
        for (int k = 0; k < MT; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            f32x4 y{o[k][4 * e], o[k][4 * e + 1], o[k][4 * e + 2], o[k][4 * e + 3]};
            const int d = 32 * k + 8 * e + 4 * kg;
            if (splits == 1)
              st4(static_cast<E*>(a.out) + at * D + d, l == 0.f ? zero4() : y * inv);
            else
              *reinterpret_cast<f32x4*>(a.ws + (at * splits + s) * D + d) = y;
          }
      }
      if (kg == 0) {
        if (splits > 1) {
          float* ml = a.ws + a.T * a.heads * splits * D + (at * splits + s) * 2;
          ml[0] = m;
          ml[1] = l;
        } else if (a.lse) {
          a.lse[at] = (m - bias + log2f(l)) * 0.693147180559945309f;
        }
      }
    }
    __syncthreads();
  }
}

template <class E, int D>
void launch_dim(const AttendArgs& a, int splits, hipStream_t st) {
  const int64_t each = (int64_t)(a.N + 1) * a.kv_heads * splits;
  const int64_t wanted = ((int64_t)a.max_queries * (a.heads / a.kv_heads) + kRows - 1) / kRows;
  const int tiles = (int)std::max<int64_t>(1, std::min<int64_t>(wanted, (1 << 23) / each));
  tile_kernel<E, D><<<(unsigned)(each * tiles), 256, 0, st>>>(a, tiles, splits);
}

template <class E>
void by_dim(const AttendArgs& a, int splits, hipStream_t st) {
  if (a.D == 64)
    launch_dim<E, 64>(a, splits, st);
  else if (a.D == 128)
    launch_dim<E, 128>(a, splits, st);
  else
    launch_dim<E, 256>(a, splits, st);
}

}  // namespace

void launch_attend_tiles(const AttendArgs& a, int splits, hipStream_t st) {
  if (a.fp16)
    by_dim<f16>(a, splits, st);
  else
    by_dim<bf16>(a, splits, st);
}

}  // namespace cqgdn
