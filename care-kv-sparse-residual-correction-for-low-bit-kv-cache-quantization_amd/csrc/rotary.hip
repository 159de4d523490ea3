// Rotary positions from the positions themselves (rotate_heads): for pair i of
// a head's first rotary_dim values and position p,
//   t = p f_i,  y1 = a (x1 cos t - x2 sin t),  y2 = a (x2 cos t + x1 sin t)
// (inverse: -t), the pairs (i, i + r/2) or (2i, 2i + 1), the other values
// copied.  q and k in one launch.
//
// Angles: p f_i / 2 pi turns in 64 bits, their distance to the nearest whole
// turn rounded to 32 (at most 2^-26 turns off), sine and cosine of that in 32
// bits.  A 32-bit product alone would be half a turn off at p f_i = 2^25.
// The products are 32 bits, rounded once to the element type.
//
// Bound by memory: each element is read and written once.  A thread owns PV
// pairs of one token and walks over heads, so that an angle is computed once
// for all the heads of the walk (64-bit products are what would cost here);
// where there are too few tokens to fill the GPU the walk is cut into shorter
// ones.
//
// Measured: 4 x 8192 tokens of 80 heads, D = 128 (1.34 GB) 259 us, 5.18 TB/s, the
// rate of a large copy (5.17); 8 x 2047 tokens of 40 heads, half of each turned
// (336 MB), 72 us, 4.7 TB/s; one token 4 us.  Stores that pass the caches made
// the first 245-250 us and the second, part of which stays in them, 83-85.
#include "common.h"
#include "host_util.h"

namespace carekv {

struct RotaryArgs {
  const char* q;
  const char* k;
  char* qo;
  char* ko;
  const void* pos;
  const double* freqs;
  long pos_batch;
  long sb[2], sh[2], st[2], ob[2], oh[2], ot[2];  // strides in bytes, q and k
  int T, D, R, Hq, H;  // H = query and kv heads together
  int heads;           // heads of a walk
  int inverse;
  float scale;
  long rows;           // batch * T
};

// N elements at p: 16-byte pieces where WIDE (the host checked the alignment), else one by one
template <typename E, int N, bool WIDE>
__device__ __forceinline__ void load_vec(E* x, const char* p) {
  if constexpr (WIDE && N * sizeof(E) % 16 == 0) {
#pragma unroll
    for (int i = 0; i < (int)(N * sizeof(E) / 16); ++i) {
      const uint4 v = *reinterpret_cast<const uint4*>(p + 16 * i);
      __builtin_memcpy(reinterpret_cast<char*>(x) + 16 * i, &v, 16);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = reinterpret_cast<const E*>(p)[i];
  }
}
template <typename E, int N, bool WIDE>
__device__ __forceinline__ void store_vec(char* p, const E* x) {
  if constexpr (WIDE && N * sizeof(E) % 16 == 0) {
#pragma unroll
    for (int i = 0; i < (int)(N * sizeof(E) / 16); ++i) {
      uint4 v;
      __builtin_memcpy(&v, reinterpret_cast<const char*>(x) + 16 * i, 16);
      *reinterpret_cast<uint4*>(p + 16 * i) = v;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) reinterpret_cast<E*>(p)[i] = x[i];
  }
}

// P64: int64 positions.  A token's threads: R / 2 / PV that rotate, then
// (D - R) / 2 / PV that copy 2 PV values each.
template <typename E, int PV, bool IL, bool P64>
__global__ __launch_bounds__(256) void rotate_heads_kernel(RotaryArgs a) {
  constexpr bool W = PV > 1;
  const int per = a.D / 2 / PV, nrot = a.R / 2 / PV;
  const uint32_t i = blockIdx.x * 256 + threadIdx.x, row = i / (uint32_t)per;  // (a grid's threads are below 2^32)
  if (row >= a.rows) return;
  const int u = (int)(i - row * per);
  const long b = row / (uint32_t)a.T, t = row - b * a.T;
  const int h0 = blockIdx.y * a.heads, h1 = min(h0 + a.heads, a.H);
  const bool rot = u < nrot;
  float c[PV], s[PV];
  if (rot) {
    const long pi = b * a.pos_batch + t;
    const double p = P64 ? (double)reinterpret_cast<const int64_t*>(a.pos)[pi]
                         : (double)reinterpret_cast<const int32_t*>(a.pos)[pi];
#pragma unroll
    for (int j = 0; j < PV; ++j) {
      const double turns = p * a.freqs[u * PV + j] * 0.15915494309189533577;  // 1 / 2 pi
      const float r = (float)(turns - rint(turns));
      sincospif(2.f * r, &s[j], &c[j]);
      s[j] *= a.inverse ? -a.scale : a.scale;
      c[j] *= a.scale;
    }
  }
  // element offsets of the thread's two runs of PV values (IL, copies: one run of 2 PV)
  const int e1 = rot ? (IL ? 2 * u * PV : u * PV) : a.R + 2 * (u - nrot) * PV;
  const int e2 = rot && !IL ? e1 + a.R / 2 : e1 + PV;
  for (int h = h0; h < h1; ++h) {
    const int isk = h >= a.Hq, hh = isk ? h - a.Hq : h;
    const char* x = (isk ? a.k : a.q) + b * a.sb[isk] + hh * a.sh[isk] + t * a.st[isk];
    char* y = (isk ? a.ko : a.qo) + b * a.ob[isk] + hh * a.oh[isk] + t * a.ot[isk];
    E v[2 * PV], w[2 * PV];
    load_vec<E, PV, W>(v, x + e1 * sizeof(E));
    load_vec<E, PV, W>(v + PV, x + e2 * sizeof(E));
    if (rot) {
#pragma unroll
      for (int j = 0; j < PV; ++j) {
        const int i1 = IL ? 2 * j : j, i2 = IL ? 2 * j + 1 : PV + j;
        const float x1 = (float)v[i1], x2 = (float)v[i2];
        w[i1] = (E)fmaf(x1, c[j], -(x2 * s[j]));
        w[i2] = (E)fmaf(x2, c[j], x1 * s[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 2 * PV; ++j) w[j] = v[j];
    }
    store_vec<E, PV, W>(y + e1 * sizeof(E), w);
    store_vec<E, PV, W>(y + e2 * sizeof(E), w + PV);
  }
}

}  // namespace carekv

using namespace carekv;

extern "C" int carekv_rotate_heads(const carekv_rotary_params* pp, const void* q, const void* k, const void* positions,
                                   const double* freqs, void* qo, void* ko, void* stream) {
  CAREKV_REQUIRE(pp, "null argument");
  const carekv_rotary_params& p = *pp;
  CAREKV_REQUIRE(p.batch >= 0 && p.seq_len >= 0 && p.n_heads >= 0 && p.n_kv_heads >= 0, "negative counts");
  CAREKV_REQUIRE(p.head_dim > 0 && p.head_dim % 2 == 0 && p.rotary_dim >= 0 && p.rotary_dim % 2 == 0 &&
                     p.rotary_dim <= p.head_dim, "head_dim and rotary_dim must be even, 0 <= rotary_dim <= head_dim");
  CAREKV_REQUIRE(p.dtype >= CAREKV_F16 && p.dtype <= CAREKV_F32, "dtype must be CAREKV_F16, CAREKV_BF16 or CAREKV_F32");
  CAREKV_REQUIRE(p.pos_bits == 32 || p.pos_bits == 64, "pos_bits must be 32 or 64");
  const long rows = (long)p.batch * p.seq_len;
  const long heads = (long)p.n_heads + p.n_kv_heads;
  if (rows == 0 || heads == 0) return CAREKV_OK;
  CAREKV_REQUIRE(heads < 65536, "too many heads");
  CAREKV_REQUIRE((p.n_heads == 0 || (q && qo)) && (p.n_kv_heads == 0 || (k && ko)) && positions &&
                     (p.rotary_dim == 0 || freqs), "null argument");
  const int es = p.dtype == CAREKV_F32 ? 4 : 2;
  RotaryArgs a{};
  a.q = (const char*)q; a.k = (const char*)k; a.qo = (char*)qo; a.ko = (char*)ko;
  a.pos = positions; a.freqs = freqs; a.pos_batch = p.pos_batch;
  a.sb[0] = p.q_sb * es; a.sh[0] = p.q_sh * es; a.st[0] = p.q_st * es;
  a.sb[1] = p.k_sb * es; a.sh[1] = p.k_sh * es; a.st[1] = p.k_st * es;
  a.ob[0] = p.qo_sb * es; a.oh[0] = p.qo_sh * es; a.ot[0] = p.qo_st * es;
  a.ob[1] = p.ko_sb * es; a.oh[1] = p.ko_sh * es; a.ot[1] = p.ko_st * es;
  uintptr_t bits = 0;
  for (int i = 0; i < 2; ++i) {
    const int h = i ? p.n_kv_heads : p.n_heads;
    if (h == 0) continue;
    bits |= operand_bits(i ? k : q, {{p.batch, a.sb[i]}, {h, a.sh[i]}, {p.seq_len, a.st[i]}});
    bits |= operand_bits(i ? ko : qo, {{p.batch, a.ob[i]}, {h, a.oh[i]}, {p.seq_len, a.ot[i]}});
  }
  a.T = p.seq_len; a.D = p.head_dim; a.R = p.rotary_dim; a.Hq = p.n_heads; a.H = (int)heads;
  a.inverse = p.inverse != 0; a.scale = p.scale; a.rows = rows;
  // 8 pairs a thread (16-byte accesses) where the sizes and every address allow it, else one
  const bool wide = (bits & 15) == 0 && p.rotary_dim % 16 == 0 && p.head_dim % 16 == 0;
  const long threads = rows * (p.head_dim / 2 / (wide ? 8 : 1));
  const long blocks = (threads + 255) / 256;
  CAREKV_REQUIRE(grid_fits(blocks, 256), "too many elements");
  // walks over all heads, cut shorter until 2048 work-groups (8 a CU) are there
  long cuts = (2048 + blocks - 1) / blocks;
  if (cuts > heads) cuts = heads;
  a.heads = (int)((heads + cuts - 1) / cuts);
  const dim3 grid((unsigned)blocks, (unsigned)((heads + a.heads - 1) / a.heads));
  hipStream_t s = (hipStream_t)stream;
  auto go = [&](auto e, auto pv) {
    using E = decltype(e);
    constexpr int PV = decltype(pv)::value;
    if (p.interleaved) {
      if (p.pos_bits == 64) hipLaunchKernelGGL((rotate_heads_kernel<E, PV, true, true>), grid, dim3(256), 0, s, a);
      else hipLaunchKernelGGL((rotate_heads_kernel<E, PV, true, false>), grid, dim3(256), 0, s, a);
    } else {
      if (p.pos_bits == 64) hipLaunchKernelGGL((rotate_heads_kernel<E, PV, false, true>), grid, dim3(256), 0, s, a);
      else hipLaunchKernelGGL((rotate_heads_kernel<E, PV, false, false>), grid, dim3(256), 0, s, a);
    }
  };
  auto typed = [&](auto pv) {
    if (p.dtype == CAREKV_F16) go(_Float16{}, pv);
    else if (p.dtype == CAREKV_BF16) go(__bf16{}, pv);
    else go(float{}, pv);
  };
  if (wide) typed(std::integral_constant<int, 8>{});
  else typed(std::integral_constant<int, 1>{});
  CAREKV_CHECK_LAUNCH("rotate_heads");
  return CAREKV_OK;
}
