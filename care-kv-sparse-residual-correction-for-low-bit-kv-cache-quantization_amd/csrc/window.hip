// Attention of (ragged) prompts and single tokens over 16-bit rows, inside a
// window and over the first tokens (window_attention):
//   o = sum_j e^(s_j) v_j / sum_j e^(s_j), s_j = scale q . k_j,
// over the keys that the row sees (rows_attn.h).
//
// Many rows: bound by the products and, with them, the exponentials, at the clock
// that the card's power allows; the main loop is tile_attn.h's, here are its tiles.
// Few rows (single tokens, a few drafts): bound by reading K and V once, and in
// short windows by the chain of latencies.
#include <algorithm>
#include <cmath>

#include "host_util.h"
#include "tile_attn.h"

namespace carekv {

struct WindowArgs : RowsArgs {
  const char* k;
  const char* v;
  long k_sb, k_sh, k_st, v_sb, v_sh, v_st;  // bytes
};

// Whether one of two elements is infinite or no number: its exponent's bits all set.
template <typename ET>
__device__ __forceinline__ uint32_t not_finite2(uint32_t x) {
  constexpr uint32_t e = std::is_same<typename ET::E, _Float16>::value ? 0x7c007c00u : 0x7f807f80u, one = e & (~e << 1);
  return ((x & e) + one) & 0x80008000u;
}

// Whether any of 2 n elements is: 0 times it, added up, is no number then.
template <typename ET, int N>
__device__ __forceinline__ bool not_finite(const uint32_t* x) {
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if constexpr (std::is_same<typename ET::E, _Float16>::value) {
      half2_t h;
      __builtin_memcpy(&h, &x[i], 4);
      sum = __builtin_amdgcn_fdot2(h, half2_t{}, sum, false);
    } else {
      typedef __bf16 bhalf2_t __attribute__((ext_vector_type(2)));
      bhalf2_t h;
      __builtin_memcpy(&h, &x[i], 4);
      sum = __builtin_amdgcn_fdot2_f32_bf16(h, bhalf2_t{}, sum, false);
    }
  }
  return !(sum == 0.f);
}

// 16-bit rows as the tiles' source.  LDS rows are padded by 32 bytes: every bank once per read pattern.
template <typename ET_, int D_>
struct Rows16 {
  using Args = WindowArgs;
  using ET = ET_;
  using Out = typename ET::E;
  using V8 = typename ET::V8;
  static constexpr int D = D_, RS = 2 * D + 32, kK = 32 * RS, kV = 32 * RS, CHR = D / 8, NCH = 32 * CHR / 256;
  typedef short short4_t __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) short4_t lds_short4;
  const char* kbase;
  const char* vbase;
  long k_st, v_st;
  int len, lane, at, next;    // keys; the thread's place in a tile of LDS; the tile to be loaded
  uint32_t k_off[NCH], v_off[NCH];
  uint32_t k[NCH][4], v[NCH][4];

  __device__ __forceinline__ Rows16(const Args& a, int b, int hk, const SeqRows& seq, int, int, int lane_)
      : kbase(a.k + b * a.k_sb + hk * a.k_sh), vbase(a.v + b * a.v_sb + hk * a.v_sh), k_st(a.k_st), v_st(a.v_st),
        len(seq.len), lane(lane_) {
    const int row = threadIdx.x / CHR, col = threadIdx.x % CHR * 16;
    at = row * RS + col;
#pragma unroll
    for (int x = 0; x < NCH; ++x) {
      k_off[x] = (uint32_t)((row + 256 / CHR * x) * k_st + col);
      v_off[x] = (uint32_t)((row + 256 / CHR * x) * v_st + col);
    }
  }
  static __device__ __forceinline__ float load_q(V8* qf, const Args& a, int b, int hk, int r, int g) {
    r = min(r, a.M - 1);
    const int t = r / a.by_g, h = hk * a.G + r - t * a.G;
    const char* qp = a.q + b * a.q_sb + h * a.q_sh + t * a.q_st;
#pragma unroll
    for (int s = 0; s < D / 32; ++s) {
      uint4 x = *reinterpret_cast<const uint4*>(qp + (32 * s + 8 * g) * 2);
      x.x = (x.x ^ a.q_sign) & a.q_keep; x.y = (x.y ^ a.q_sign) & a.q_keep;
      x.z = (x.z ^ a.q_sign) & a.q_keep; x.w = (x.w ^ a.q_sign) & a.q_keep;
      __builtin_memcpy(&qf[s], &x, 16);
    }
    return a.sm_log2;
  }
  // a tile is a buffer resource of its rows, a thread's offsets in it stay the same; rows past the length read zeros
  static __device__ __forceinline__ void load(uint32_t (&x)[NCH][4], const char* base, long st, const uint32_t (&off)[NCH],
                                              int j0, int len) {
    const __amdgpu_buffer_rsrc_t r = make_rsrc(base + (long)j0 * st, (uint32_t)((min(32, len - j0) - 1) * st + 2 * D));
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const auto u = __builtin_amdgcn_raw_buffer_load_b128(r, off[i], 0, 0);
      x[i][0] = u[0]; x[i][1] = u[1]; x[i][2] = u[2]; x[i][3] = u[3];
    }
  }
  __device__ __forceinline__ void look(int tile) { next = tile; }
  __device__ __forceinline__ void load() {
    load(k, kbase, k_st, k_off, 32 * next, len);
    load(v, vbase, v_st, v_off, 32 * next, len);
  }
  template <bool CARE>
  __device__ __forceinline__ bool store(char* kb, char* vb, int) {
    bool odd = false;
    if constexpr (CARE) {
#pragma unroll
      for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint32_t u = not_finite2<ET>(v[i][x]);
          odd |= u != 0;
          v[i][x] &= (u & 0x8000u ? 0u : 0xffffu) | (u >> 31 ? 0u : 0xffff0000u);
        }
    }
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      *reinterpret_cast<uint4*>(kb + at + 256 / CHR * i * RS) = make_uint4(k[i][0], k[i][1], k[i][2], k[i][3]);
      *reinterpret_cast<uint4*>(vb + at + 256 / CHR * i * RS) = make_uint4(v[i][0], v[i][1], v[i][2], v[i][3]);
    }
    return odd;
  }
  __device__ __forceinline__ V8 k_op(const char* buf, int tt, int ks) const {
    V8 r;
    *reinterpret_cast<uint4*>(&r) = *reinterpret_cast<const uint4*>(buf + (16 * tt + (lane & 15)) * RS + (32 * ks + 8 * (lane >> 4)) * 2);
    return r;
  }
  __device__ __forceinline__ V8 v_op(const char* buf, int dt) const {
    const __attribute__((address_space(3))) char* row = (const __attribute__((address_space(3))) char*)buf +
                                                        (4 * (lane >> 4) + ((lane & 15) >> 2)) * RS + (lane & 3) * 8;
    const short4_t v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(row + 32 * dt));
    const short4_t v2 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(row + 16 * RS + 32 * dt));
    V8 r;
    __builtin_memcpy(&r, &v1, 8);
    __builtin_memcpy(reinterpret_cast<char*>(&r) + 8, &v2, 8);
    return r;
  }
  __device__ __forceinline__ int there() const { return 3; }
  // from where they came: with a weight over 0 they are the result whatever it is
  template <int NQ, int DT>
  __device__ __forceinline__ void odd_values(const Args& a, float4_t (&o)[NQ][DT], const RowSight (&sight)[NQ], int tile) const {
    const int j0 = 32 * tile;
#pragma unroll 1
    for (int key = 0; key < min(32, len - j0); ++key) {
      const char* src = vbase + (long)(j0 + key) * v_st + 8 * (lane >> 4);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        asm volatile("" ::: "memory");  // (one at a time: in flight together they would cost the loop its registers)
        uint32_t x[2];
        __builtin_memcpy(x, __builtin_assume_aligned(src + 32 * dt, 8), 8);
        if (!(not_finite2<ET>(x[0]) | not_finite2<ET>(x[1]))) continue;
        Out e[4];
        __builtin_memcpy(e, x, 8);
#pragma unroll
        for (int qb = 0; qb < NQ; ++qb) {
          RowSight row = sight[qb];
          row.stay_here();
#pragma unroll
          for (int y = 0; y < 4; ++y)
            if (row.sees(a, j0 + key) && !(fabsf((float)e[y]) < INFINITY)) o[qb][dt][y] += (float)e[y];
        }
      }
    }
  }
};

// Up to 32 rows of a kv head: the four waves of a work-group have the same rows and
// 32 keys each of a tile of 128, and are joined in LDS at the end.  One tile of LDS:
// the next one's rows are on their way in registers.  16 rows of 32 / 8 heads, D = 128,
// on 4097 keys (268 MB): 48 us, 5.6 TB/s; one row of 32 / 4 heads, D = 64, through a
// window of 1024 in a graph 8.6 us, two launches.
template <typename ET, int D>
__global__ __launch_bounds__(256, 2) void window_few_kernel(WindowArgs a) {
  using V8 = typename ET::V8;
  using E = typename ET::E;
  constexpr int NT = 256, WK = 4, KT = 32 * WK, TT = 2, NQ = 2, QB = 16 * NQ;
  constexpr int KRS = 2 * D + 32, VRS = 2 * D + 32;  // padded LDS rows: every bank once per read pattern
  constexpr int KS = D / 32, DT = D / 16, CHR = D / 8, NCH = 2 * KT * CHR / NT;
  constexpr int KBUF = KT * KRS, BUF = KBUF + KT * VRS;
  __shared__ __align__(16) char lds[BUF];
  __shared__ int s_odd;  // whether a tile held a V value that is not finite
  typedef short short4_t __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) short4_t lds_short4;

  const int it = xcd_item(a);
  const int sp_blk = it / a.by_nsplit, sp = it - sp_blk * a.nsplit;
  const int bh = sp_blk / a.by_nqb, qblk = a.nqb - 1 - (sp_blk - bh * a.nqb);  // (blocks with more keys first)
  const int b = bh / a.by_hkv, hk = bh - b * a.Hkv;
  const int lane = threadIdx.x & 63;
  const int wk = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // the wave, and its share of the keys
  const int g = lane >> 4, c16 = lane & 15;
  const SeqRows seq(a, b);
  const int r0 = qblk * QB, t0 = r0 / a.by_g, t1 = (min(r0 + QB, a.M) - 1) / a.by_g + 1;
  const Span<KT> span(a, seq, t0, t1);
  const Span<32> mine(a, seq, t0, t1);
  const int i0 = sp * a.tps, i1 = min(i0 + a.tps, span.n), nt = i1 - i0;
  if (a.nsplit > 1 && nt <= 0) return;  // (the join does not read it)
  const char* kbase = a.k + b * a.k_sb + hk * a.k_sh;
  const char* vbase = a.v + b * a.v_sb + hk * a.v_sh;

  // Q^T operands: sub-block qb, step s -> row r0 + 16 qb + c16, dims 32s + 8g ..; negated for a negative scale
  V8 qf[NQ][KS];
  RowSight sight[NQ];
#pragma unroll
  for (int qb = 0; qb < NQ; ++qb) {
    sight[qb] = RowSight(a, seq, r0 + 16 * qb + c16);
    const int r = min(r0 + 16 * qb + c16, a.M - 1), t = r / a.by_g, h = hk * a.G + r - t * a.G;
    const char* qp = a.q + b * a.q_sb + h * a.q_sh + t * a.q_st;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      uint4 v = *reinterpret_cast<const uint4*>(qp + (32 * s + 8 * g) * 2);
      v.x = (v.x ^ a.q_sign) & a.q_keep; v.y = (v.y ^ a.q_sign) & a.q_keep;
      v.z = (v.z ^ a.q_sign) & a.q_keep; v.w = (v.w ^ a.q_sign) & a.q_keep;
      __builtin_memcpy(&qf[qb][s], &v, 16);
    }
  }

  uint32_t stg[NCH][4];
  const int srow = threadIdx.x / CHR, scol = threadIdx.x % CHR * 16;  // (chunk k: row srow + NT / CHR k of K, then V)
  uint32_t off[NCH];
#pragma unroll
  for (int k = 0; k < NCH; ++k)
    off[k] = (uint32_t)((srow + NT / CHR * (k % (NCH / 2))) * (k < NCH / 2 ? a.k_st : a.v_st) + scol);
  // A tile is a buffer resource of its rows, a thread's offsets in it stay the same; rows past the length read zeros.
  auto load_tile = [&](int i) {
    const int j0 = span.tile(i0 + i) * KT, last = min(KT, seq.len - j0) - 1;
    const __amdgpu_buffer_rsrc_t rk = make_rsrc(kbase + (long)j0 * a.k_st, (uint32_t)(last * a.k_st + 2 * D));
    const __amdgpu_buffer_rsrc_t rv = make_rsrc(vbase + (long)j0 * a.v_st, (uint32_t)(last * a.v_st + 2 * D));
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const auto v = __builtin_amdgcn_raw_buffer_load_b128(k < NCH / 2 ? rk : rv, off[k], 0, 0);
      stg[k][0] = v[0]; stg[k][1] = v[1]; stg[k][2] = v[2]; stg[k][3] = v[3];
    }
  };
  // (a weight of 0 times a value that is not finite would be no number: such a value is 0 in the tile, and added at the
  // end to the rows that see it)
  auto store_tile = [&] {
    if (__builtin_expect(not_finite<ET, 2 * NCH>(&stg[NCH / 2][0]), 0)) {
      s_odd = 1;
#pragma unroll
      for (int k = NCH / 2; k < NCH; ++k)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint32_t n = not_finite2<ET>(stg[k][x]);
          stg[k][x] &= (n & 0x8000u ? 0u : 0xffffu) | (n >> 31 ? 0u : 0xffff0000u);
        }
    }
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int row = srow + NT / CHR * (k % (NCH / 2));
      char* dst = lds + (k < NCH / 2 ? row * KRS : KBUF + row * VRS) + scol;
      *reinterpret_cast<uint4*>(dst) = make_uint4(stg[k][0], stg[k][1], stg[k][2], stg[k][3]);
    }
  };

  float m_run[NQ], l_run[NQ];
  float4_t o[NQ][DT];
#pragma unroll
  for (int qb = 0; qb < NQ; ++qb) {
    m_run[qb] = kLowest;
    l_run[qb] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[qb][dt] = float4_t{0.f, 0.f, 0.f, 0.f};
  }
  const float c = a.sm_log2;  // (not negative)
  if (threadIdx.x == 0) s_odd = 0;
  __syncthreads();
  if (nt > 0) {
    load_tile(0);
    store_tile();
  }
  __syncthreads();
  if (nt > 1) load_tile(1);
  for (int i = 0; i < nt; ++i) {
    const int jw = span.tile(i0 + i) * KT + 32 * wk;  // the wave's first key of the tile
    const char* kb = lds + 32 * wk * KRS;
    const char* vb = lds + KBUF + 32 * wk * VRS;
    if (mine.n > 0 && jw <= mine.hi && (jw + 31 > mine.first - a.window || jw < a.sink)) {
      // (raised wave priority over the products: a wave with products to issue goes before others' softmax)
      __builtin_amdgcn_s_setprio(1);
      float4_t s[TT][NQ];
#pragma unroll
      for (int tt = 0; tt < TT; ++tt) {
#pragma unroll
        for (int qb = 0; qb < NQ; ++qb) s[tt][qb] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          V8 ak;
          *reinterpret_cast<uint4*>(&ak) = *reinterpret_cast<const uint4*>(kb + (16 * tt + c16) * KRS + (32 * ks + 8 * g) * 2);
#pragma unroll
          for (int qb = 0; qb < NQ; ++qb) s[tt][qb] = ET::mfma(ak, qf[qb][ks], s[tt][qb]);
        }
      }
      __builtin_amdgcn_s_setprio(0);
      if (!mine.whole(a, jw)) {
#pragma unroll
        for (int qb = 0; qb < NQ; ++qb) {
          RowSight row = sight[qb];
          row.stay_here();
#pragma unroll
          for (int tt = 0; tt < TT; ++tt)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (!row.sees(a, jw + 16 * tt + 4 * g + k)) s[tt][qb][k] = -INFINITY;
        }
      }
      // base-2 logits x = c s folded into the exponent: max x = c max s, e^.. = 2^fma(s, c, -reference)
      float mx[NQ];
      bool any_over = false, over[NQ];
#pragma unroll
      for (int qb = 0; qb < NQ; ++qb) {
        mx[qb] = -INFINITY;
#pragma unroll
        for (int k = 0; k < 8; k += 2) mx[qb] = fmaxf(fmaxf(mx[qb], s[k / 4][qb][k % 4]), s[k / 4][qb][k % 4 + 1]);
        over[qb] = fmaf(mx[qb], c, -ET::kUp) > m_run[qb];
        any_over |= over[qb];
      }
      if (__any(any_over)) {
#pragma unroll
        for (int qb = 0; qb < NQ; ++qb) {
          if (!__any(over[qb])) continue;  // columns that keep their reference get a factor of exactly 1
          const float m_new = fmaxf(m_run[qb], fmaf(col_max(mx[qb]), c, -ET::kUp));
          const float f = __builtin_amdgcn_exp2f(m_run[qb] - m_new);
          m_run[qb] = m_new;
          l_run[qb] *= f;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) o[qb][dt] *= f;
        }
      }
      V8 bp[NQ];
#pragma unroll
      for (int qb = 0; qb < NQ; ++qb) {
        float ls = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float p = __builtin_amdgcn_exp2f(fmaf(s[k / 4][qb][k % 4], c, -m_run[qb]));
          ls += p;
          bp[qb][k] = (E)p;
        }
        l_run[qb] += ls;
      }
      const __attribute__((address_space(3))) char* vrow =
          (const __attribute__((address_space(3))) char*)vb + (4 * g + (c16 >> 2)) * VRS + (c16 & 3) * 8;
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const short4_t v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(vrow + 32 * dt));
        const short4_t v2 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(vrow + 16 * VRS + 32 * dt));
        V8 av;
        __builtin_memcpy(&av, &v1, 8);
        __builtin_memcpy(reinterpret_cast<char*>(&av) + 8, &v2, 8);
#pragma unroll
        for (int qb = 0; qb < NQ; ++qb) o[qb][dt] = ET::mfma(av, bp[qb], o[qb][dt]);
      }
    }
    __builtin_amdgcn_s_setprio(0);
    __syncthreads();
    if (i + 1 < nt) store_tile();
    if (i + 2 < nt) load_tile(i + 2);
    __syncthreads();
  }
  // Values that are not finite, from where they came, into the rows that see them: with a weight over 0 they are the
  // result whatever it is, so that they are added when no sum is rescaled any more.
  const bool odd = s_odd;
  if (__builtin_expect(odd, 0)) {
#pragma unroll 1
    for (int i = 0; i < nt; ++i) {
      const int jw = span.tile(i0 + i) * KT + 32 * wk, keys = min(32, seq.len - jw);
      bool some = false;
      for (int x = lane; x < keys * CHR; x += 64) {
        uint32_t u[4];
        __builtin_memcpy(u, __builtin_assume_aligned(vbase + (long)(jw + x / CHR) * a.v_st + x % CHR * 16, 16), 16);
        some |= not_finite<ET, 4>(u);
      }
      if (!__any(some)) continue;
#pragma unroll 1
      for (int key = 0; key < keys; ++key) {
        const char* src = vbase + (long)(jw + key) * a.v_st + 8 * g;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          asm volatile("" ::: "memory");  // (one at a time: in flight together they would cost the loop its registers)
          uint32_t x[2];
          __builtin_memcpy(x, __builtin_assume_aligned(src + 32 * dt, 8), 8);
          if (!(not_finite2<ET>(x[0]) | not_finite2<ET>(x[1]))) continue;
          E v[4];
          __builtin_memcpy(v, x, 8);
#pragma unroll
          for (int qb = 0; qb < NQ; ++qb)
#pragma unroll
            for (int y = 0; y < 4; ++y)
              if (sight[qb].sees(a, jw + key) && !(fabsf((float)v[y]) < INFINITY)) o[qb][dt][y] += (float)v[y];
        }
      }
    }
  }
  float lt[NQ];
#pragma unroll
  for (int qb = 0; qb < NQ; ++qb) lt[qb] = col_sum(l_run[qb]);
  // the waves' parts of the same rows: (m, l) of every wave, then O scaled to the joint maximum, 16 rows at a time
  // in the tiles' LDS, added in wave order; a wave keeps the dims of tiles wk, wk + WK ..
  __shared__ float s_ml[WK][QB][2];
  float* so = reinterpret_cast<float*>(lds);  // [waves][DT][64 lanes][4]
  static_assert(WK * DT * 1024 <= BUF, "the waves' O fits the tiles' LDS");
#pragma unroll
  for (int qb = 0; qb < NQ; ++qb)
    if (g == 0) { s_ml[wk][16 * qb + c16][0] = m_run[qb]; s_ml[wk][16 * qb + c16][1] = lt[qb]; }
  __syncthreads();
#pragma unroll
  for (int qb = 0; qb < NQ; ++qb) {
    float m = kLowest, l = 0.f;
#pragma unroll
    for (int i = 0; i < WK; ++i) m = fmaxf(m, s_ml[i][16 * qb + c16][0]);
#pragma unroll
    for (int i = 0; i < WK; ++i) l += s_ml[i][16 * qb + c16][1] * __builtin_amdgcn_exp2f(s_ml[i][16 * qb + c16][0] - m);
    const float f = __builtin_amdgcn_exp2f(m_run[qb] - m);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      *reinterpret_cast<float4_t*>(so + ((wk * DT + dt) * 64 + lane) * 4) = odd ? rescaled(o[qb][dt], f) : o[qb][dt] * f;
    m_run[qb] = m;
    lt[qb] = l;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < (DT + WK - 1) / WK; ++u) {
      const int dt = wk + WK * u;
      if (dt >= DT) break;
      float4_t v = *reinterpret_cast<const float4_t*>(so + (dt * 64 + lane) * 4);
#pragma unroll
      for (int i = 1; i < WK; ++i) v += *reinterpret_cast<const float4_t*>(so + ((i * DT + dt) * 64 + lane) * 4);
      o[qb][u] = v;
    }
    __syncthreads();
  }
  // the rows' results, or the split's partial (lane: row r0 + 16qb + c16, dims 16dt + 4g ..)
  constexpr int OT = (DT + WK - 1) / WK;
#pragma unroll
  for (int qb = 0; qb < NQ; ++qb) {
    const int r = r0 + 16 * qb + c16;
    if (r >= a.M) continue;
    const bool first = g == 0 && wk == 0;
    if (a.nsplit == 1) {
      const bool pad = sight[qb].top < 0;  // (what a row of padding holds is not used)
      const float l = pad ? 0.f : lt[qb];
      char* row = out_row(a, b, hk, r);
#pragma unroll
      for (int u = 0; u < OT; ++u)
        if (wk + WK * u < DT) write4<E>(a, row, 16 * (wk + WK * u) + 4 * g, pad ? float4_t{0.f, 0.f, 0.f, 0.f} : o[qb][u], l);
      if (a.lse && first) write_lse(a, b, hk, r, m_run[qb], l);
    } else {
      const long pr = (long)sp * a.rows + (long)bh * a.M + r;
      float* dst = a.po + pr * D + 4 * g;
#pragma unroll
      for (int u = 0; u < OT; ++u)
        if (wk + WK * u < DT) *reinterpret_cast<float4_t*>(dst + 16 * (wk + WK * u)) = o[qb][u];
      if (first) {
        a.pml[2 * pr] = m_run[qb];
        a.pml[2 * pr + 1] = lt[qb];
      }
    }
  }
}

namespace {
// How a call is cut: at most 32 rows a kv head share the work-group's waves by
// keys (wq = 1, wk = 4, tiles of 128 keys), more by rows (wq = 4, wk = 1, 32 keys).
// Few rows: key splits until 512 work-groups (2 a CU) are there, down to a tile
// each, at most 32 for the join's sake, and none up to 512 keys (D = 128: 256), where
// the join's launch costs the host more than they save; us a call, by splits: 32 / 4 heads, D = 64,
// on 1000 keys 1 / 4 / 8: 12.9 / 8.9 / 8.1, on 4097 4 / 8 / 16 / 32: 16.6 / 12.5 / 10.7 /
// 10.3; 16 x 32 / 8 heads, D = 128, on 4097 2 / 4 / 8 / 16: 47.9 / 46.9 / 48.4 / 50.9.  Many:
// best_splits.
struct WindowPlan {
  int wq, wk, nqb, nsplit, tps;
};
WindowPlan window_plan(const carekv_window_params& p) {
  WindowPlan r{};
  const long M = (long)p.seq_len * (p.n_heads / p.n_kv_heads);
  r.wq = M <= 32 ? 1 : 4;
  r.wk = M <= 32 ? 4 : 1;
  r.nqb = (int)((M + 32 * r.wq - 1) / (32 * r.wq));
  const int kt = 32 * r.wk;
  long keys = p.n_keys;  // that a block of rows may see
  if (p.window > 0) keys = std::min(keys, (long)p.window + std::min<long>(p.seq_len, 32L * r.wq) + p.sink + 2 * kt);
  const long tiles = std::max(1L, (keys + kt - 1) / kt), wgs = std::max(1L, (long)p.batch * p.n_kv_heads * r.nqb);
  const double mean = std::min((double)tiles, mean_keys(p.n_keys, p.seq_len, keys) / kt + 1);
  const long ns = r.wq == 4 ? best_splits(tiles, mean, wgs, (long)p.batch * p.seq_len * p.n_heads, p.head_dim)
                  : tiles * p.head_dim <= 4 * 64 ? 1 : std::max(1L, std::min(std::min(32L, 512 / wgs), tiles));
  r.tps = (int)((tiles + ns - 1) / ns);
  r.nsplit = (int)((tiles + r.tps - 1) / r.tps);
  return r;
}
long window_ws(const carekv_window_params& p, const WindowPlan& r) {
  const long rows = (long)p.batch * p.seq_len * p.n_heads;
  return r.nsplit > 1 ? r.nsplit * rows * (2 + p.head_dim) * 4 : 0;
}
int check_window(const carekv_window_params* pp) {
  CAREKV_REQUIRE(pp, "null argument");
  const carekv_window_params& p = *pp;
  CAREKV_REQUIRE(p.head_dim == 64 || p.head_dim == 128, "head_dim must be 64 or 128");
  CAREKV_REQUIRE(p.dtype == CAREKV_F16 || p.dtype == CAREKV_BF16, "dtype must be CAREKV_F16 or CAREKV_BF16");
  CAREKV_REQUIRE(p.batch >= 0 && p.seq_len >= 0 && p.n_keys >= 0 && p.window >= 0 && p.sink >= 0, "negative counts");
  CAREKV_REQUIRE(p.n_heads > 0 && p.n_kv_heads > 0 && p.n_heads % p.n_kv_heads == 0,
                 "n_heads must be a positive multiple of n_kv_heads");
  CAREKV_REQUIRE((long)p.batch * p.seq_len * p.n_heads < (1L << 30), "too many rows");
  CAREKV_REQUIRE(p.n_keys < kMaxPos && p.seq_len < kMaxPos, "n_keys and seq_len must be below 2^29");
  CAREKV_REQUIRE(p.n_keys < 2 || (p.k_st >= 0 && p.v_st >= 0 && p.k_st < (1 << 22) && p.v_st < (1 << 22)),
                 "K and V row strides must be in 0 .. 2^22 elements");
  return CAREKV_OK;
}
}  // namespace

}  // namespace carekv

using namespace carekv;

extern "C" int64_t carekv_window_attn_workspace_bytes(const carekv_window_params* pp) {
  if (check_window(pp) != CAREKV_OK) return -1;
  return window_ws(*pp, window_plan(*pp));
}

extern "C" int carekv_window_attn(const carekv_window_params* pp, const void* q, const void* k, const void* v,
                                  const int32_t* lengths, const int32_t* q_lengths, const int32_t* q_start, void* out,
                                  float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = check_window(pp);
  if (rc != CAREKV_OK) return rc;
  const carekv_window_params& p = *pp;
  const long rows = (long)p.batch * p.seq_len * p.n_heads;
  if (rows == 0) return CAREKV_OK;
  const WindowPlan plan = window_plan(p);
  CAREKV_REQUIRE(q && out && (p.n_keys == 0 || (k && v)) && (workspace || plan.nsplit < 2), "null argument");
  const uintptr_t bits = operand_bits(q, {{p.batch, 2 * p.q_sb}, {p.n_heads, 2 * p.q_sh}, {p.seq_len, 2 * p.q_st}}) |
                         operand_bits(k, {{p.batch, 2 * p.k_sb}, {p.n_kv_heads, 2 * p.k_sh}, {p.n_keys, 2 * p.k_st}}) |
                         operand_bits(v, {{p.batch, 2 * p.v_sb}, {p.n_kv_heads, 2 * p.v_sh}, {p.n_keys, 2 * p.v_st}}) |
                         (uintptr_t)workspace;
  CAREKV_REQUIRE((bits & 15) == 0, "q, k and v rows must be 16-byte aligned");
  if (workspace_bytes < window_ws(p, plan)) {
    set_error("carekv_window_attn: workspace too small (%lld < %lld)", (long long)workspace_bytes, (long long)window_ws(p, plan));
    return CAREKV_ESPACE;
  }
  WindowArgs a{};
  a.q = (const char*)q; a.k = (const char*)k; a.v = (const char*)v; a.out = (char*)out; a.lse = lse;
  a.lengths = lengths; a.q_lengths = q_lengths; a.q_start = q_start;
  a.q_sb = 2 * p.q_sb; a.q_sh = 2 * p.q_sh; a.q_st = 2 * p.q_st; a.o_sb = 2 * p.out_sb; a.o_sh = 2 * p.out_sh; a.o_st = 2 * p.out_st;
  a.k_sb = 2 * p.k_sb; a.k_sh = 2 * p.k_sh; a.k_st = 2 * p.k_st; a.v_sb = 2 * p.v_sb; a.v_sh = 2 * p.v_sh; a.v_st = 2 * p.v_st;
  a.Hq = p.n_heads; a.Hkv = p.n_kv_heads; a.G = p.n_heads / p.n_kv_heads; a.T = p.seq_len; a.M = a.G * p.seq_len;
  a.rows = rows; a.max_keys = p.n_keys;
  a.window = p.window > 0 ? std::min(p.window, 2 * kMaxPos) : 2 * kMaxPos;
  a.sink = p.sink;
  a.nqb = plan.nqb; a.nsplit = plan.nsplit; a.tps = plan.tps; a.qb_rows = 32 * plan.wq;
  a.by_g = FastDiv(a.G); a.by_nqb = FastDiv(a.nqb); a.by_hkv = FastDiv(a.Hkv); a.by_nsplit = FastDiv(a.nsplit); a.by_m = FastDiv(a.M);
  set_groups(a, (long)a.nqb * a.nsplit, (long)p.batch * a.Hkv);
  a.po = (float*)workspace;
  a.pml = a.po + plan.nsplit * rows * p.head_dim;
  set_scale(a, p.sm_scale);
  set_period(a, p.window, (a.qb_rows + a.G - 1) / a.G, 32 * plan.wk);
  set_alignment(a, p.batch);
  hipStream_t s = (hipStream_t)stream;
  const long wgs = (long)p.batch * a.Hkv * a.nqb * a.nsplit;
  CAREKV_REQUIRE(grid_fits(wgs, 256) && grid_fits(rows / (256 / p.head_dim) + 1, 256), "too many rows");
  return dispatch_elem_d(p.dtype, p.head_dim, [&](auto et, auto d) {
    using ET = decltype(et);
    constexpr int D = decltype(d)::value;
    const dim3 grid((unsigned)wgs), block(256);
    if (plan.wq == 1) hipLaunchKernelGGL((window_few_kernel<ET, D>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((tile_attn_kernel<Rows16<ET, D>>), grid, block, 0, s, a);
    CAREKV_CHECK_LAUNCH("window_attn");
    if (a.nsplit > 1) {
      if (plan.wk == 4) launch_join<typename ET::E, D, 128>(a, s);
      else launch_join<typename ET::E, D, 32>(a, s);
      CAREKV_CHECK_LAUNCH("rows_join");
    }
    return CAREKV_OK;
  });
}
