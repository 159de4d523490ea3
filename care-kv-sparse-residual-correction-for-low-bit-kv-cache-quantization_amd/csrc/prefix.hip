// Attention over a prefix that every row of a batch shares (prefix_attention):
//   s_j = scale q . k_j,  o = sum_j e^(s_j) v_j / sum_j e^(s_j) over the P
// prefix rows, joined with each row's attention over tokens of its own, given
// as (o_own, lse_own):  w = e^(lse), o = (w_p o_p + w_own o_own) / (w_p + w_own).
//
// The rows of a kv head -- every sequence's, query head's and query token's of
// its group -- are one tall matrix, so a K/V tile is read once for 128 of them
// instead of once a sequence.  A work-group has 128 rows (4 waves of 32) and a
// range of the keys, flash style: K and V tiles of 32 keys in LDS (double
// buffered, one barrier a tile), S^T = K Q^T and O^T += V^T P^T on
// v_mfma_f32_16x16x32, the softmax over a query's column in 32 bits on base-2
// logits; the weights are rounded to the element type for the second product
// and their sum is not: each is off by half a step at most (2^-11 or 2^-8 of
// it).  A row's reference is its maximum less 15 in fp16, so that weights are
// up to 2^15: with the maximum itself those below 2^-14 would be subnormal and
// those below 2^-25 zero, and a long tail under one key would be lost from the
// result but not from the sum.  What is subnormal now is off by 2^-40 of the
// largest.  The keys are split over work-groups until the GPU is
// full; prefix_join_kernel then joins the splits' (reference, sum, O), kept in
// 32 bits, and the row's own part.  One split joins its own part itself.
//
// K and V rows are padded by 32 bytes in LDS: 16-byte reads of 16 rows then take
// 5.6 cycles a wave, padded by 16 bytes 9.0.
//
// Measured: 16 x 128 rows, 40 heads, D = 128, 4097 keys (172 GFLOP) 206 us, 0.83
// PFLOP/s (in bursts after a pause 217): 640 equal work-groups on 768 places, products and exponentials
// overlapping in part.  64 rows x 32 / 8 heads on 32768 keys (34 GFLOP, 134 MB
// of K and V) 55 us + 6 us for the join: 16 splits of three sets of waves, whose
// partials are 17 MB; without the sets 48 splits and 50 MB 53 + 11, 32 splits 57 +
// 9, 16 splits 71 + 6.  4 x 8 rows a head on 1000 keys 12 us, one
// launch.
#include <algorithm>
#include <cmath>

#include "fast_div.h"
#include "host_util.h"
#include "mfma16.h"

namespace carekv {

struct PrefixArgs {
  const char* q;
  const char* k;
  const char* v;
  const char* own;       // the rows' own outputs, or null
  const float* own_lse;  // [B][Hq][T]
  char* out;
  float* lse;            // [B][Hq][T], or null
  float* pml;            // [nsplit][rows][2] reference (base 2), sum
  float* po;             // [nsplit][rows][D]
  long q_sb, q_sh, q_st, k_sh, k_st, v_sh, v_st, o_sb, o_sh, o_st, w_sb, w_sh, w_st;  // bytes
  long rows;             // n_kv_heads * M
  int B, Hq, Hkv, G, T, P, M, nqb, nsplit;
  FastDiv by_t, by_g, by_nqb, by_nsplit, by_m;
  float sm_log2;         // |scale| log2(e), 1 where that is 0
  uint32_t q_sign;       // sign bits of two elements where the scale is negative
  uint32_t q_keep;       // 0 where the scale is 0 (0 times the -inf of a masked score would be NaN), else all bits
  int al8;               // rows of out and own on 8 bytes
};

// Row r of kv head hk: sequence, query head, query token.
struct PrefixRow {
  int b, h, t;
};
__device__ __forceinline__ PrefixRow prefix_row(const PrefixArgs& a, int hk, int r) {
  PrefixRow x;
  const int bg = r / a.by_t;
  x.t = r - bg * a.T;
  x.b = bg / a.by_g;
  x.h = hk * a.G + bg - x.b * a.G;
  return x;
}

// The row's own part, joined with the prefix's (m, L, O unnormalised) in 32
// bits: four dims' results, and the log-sum-exp.  A row that sees nothing (no
// prefix, lse_own = -inf) is zero with a log-sum-exp of -inf, whatever its own
// output holds.
template <typename ET>
struct PrefixOwn {
  using E = typename ET::E;
  float lo, m, f, fo;  // own log-sum-exp (base 2), joint reference, factors of the prefix's and the own part
  __device__ __forceinline__ PrefixOwn(const PrefixArgs& a, const PrefixRow& x, float mp) {
    lo = a.own ? a.own_lse[((long)x.b * a.Hq + x.h) * a.T + x.t] * kLog2e : -INFINITY;
    m = fmaxf(lo, mp);
    f = __builtin_amdgcn_exp2f(mp - m);
    fo = lo == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(lo - m);  // (NaN goes on as NaN)
  }
  // dims d .. d+3 of the row (o, l: the prefix's sums), to out
  __device__ __forceinline__ void write(const PrefixArgs& a, const PrefixRow& x, int d, float4_t o, float l) const {
    const float L = f * l + fo;
    o *= f;
    if (lo != -INFINITY) {
      const E* p = reinterpret_cast<const E*>(a.own + x.b * a.w_sb + x.h * a.w_sh + x.t * a.w_st) + d;
      E v[4];
      if (a.al8) __builtin_memcpy(v, __builtin_assume_aligned(p, 8), 8);
      else
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = p[i];
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = fmaf(fo, (float)v[i], o[i]);
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    E* dst = reinterpret_cast<E*>(a.out + x.b * a.o_sb + x.h * a.o_sh + x.t * a.o_st) + d;
    E w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (E)(o[i] * inv);
    if (a.al8) __builtin_memcpy(__builtin_assume_aligned(dst, 8), w, 8);
    else
#pragma unroll
      for (int i = 0; i < 4; ++i) dst[i] = w[i];
  }
  __device__ __forceinline__ void write_lse(const PrefixArgs& a, const PrefixRow& x, float l) const {
    const float L = f * l + fo;
    a.lse[((long)x.b * a.Hq + x.h) * a.T + x.t] = L == 0.f ? -INFINITY : (m + __log2f(L)) * kLn2;
  }
};

// WQ waves have 32 rows each, WK sets of them 32 keys of the tile each, joined
// in LDS at the end: with WQ = 1, WK = 4 few rows still use every wave, with WK =
// 3 three sets write one partial.
template <typename ET, int D, int WQ, int WK>
__global__ __launch_bounds__(64 * WQ * WK, WQ == 4 ? 3 : 2) void prefix_attn_kernel(PrefixArgs a) {
  using V8 = typename ET::V8;
  using E = typename ET::E;
  constexpr int NT = 64 * WQ * WK, KT = 32 * WK, TT = 2, NQ = 2, QW = 16 * NQ, QB = WQ * QW;
  constexpr int KRS = 2 * D + 32, VRS = 2 * D + 32;  // padded LDS rows: every bank once per read pattern
  constexpr int KS = D / 32, DT = D / 16, CHR = D / 8, NCH = 2 * KT * CHR / NT;
  constexpr int KBUF = KT * KRS, BUF = KBUF + KT * VRS, NBUF = WQ == 4 ? 2 : 1;
  __shared__ __align__(16) char lds[NBUF * BUF];
  typedef short short4_t __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) short4_t lds_short4;

  // An XCD takes consecutive items, row blocks of one (head, split) next to
  // each other: they meet in its L2.
  const int n = gridDim.x;
  int it = blockIdx.x;
  if (n % 8 == 0) it = it % 8 * (n / 8) + it / 8;
  const int blk = it / a.by_nqb, qblk = it - blk * a.nqb, hk = blk / a.by_nsplit, sp = blk - hk * a.nsplit;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c16 = lane & 15;
  const int wq = w % WQ, wk = w / WQ, r0 = qblk * QB + QW * wq;  // the wave's share of rows and keys, its first row
  const int tiles = (a.P + KT - 1) / KT;
  const int tile0 = part_start(tiles, sp, a.by_nsplit), tile1 = part_start(tiles, sp + 1, a.by_nsplit);
  const int j0 = tile0 * KT, keys = min(tile1 * KT, a.P) - j0;  // the split's keys (at least one)
  const char* kbase = a.k + hk * a.k_sh + j0 * a.k_st;
  const char* vbase = a.v + hk * a.v_sh + j0 * a.v_st;

  // Q^T operands: sub-block qb, step s -> row r0 + 16 qb + c16, dims 32s + 8g ..; negated for a negative scale
  V8 qf[NQ][KS];
#pragma unroll
  for (int qb = 0; qb < NQ; ++qb) {
    const PrefixRow x = prefix_row(a, hk, min(r0 + 16 * qb + c16, a.M - 1));
    const char* qp = a.q + x.b * a.q_sb + x.h * a.q_sh + x.t * a.q_st;
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
  // A tile is a buffer resource of its rows, a thread's offsets in it stay the same; rows past the split read zeros.
  auto load_tile = [&](int j) {
    const int last = min(KT, keys - j * KT) - 1;
    const __amdgpu_buffer_rsrc_t rk = make_rsrc(kbase + (long)j * KT * a.k_st, (uint32_t)(last * a.k_st + 2 * D));
    const __amdgpu_buffer_rsrc_t rv = make_rsrc(vbase + (long)j * KT * a.v_st, (uint32_t)(last * a.v_st + 2 * D));
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const auto v = __builtin_amdgcn_raw_buffer_load_b128(k < NCH / 2 ? rk : rv, off[k], 0, 0);
      stg[k][0] = v[0]; stg[k][1] = v[1]; stg[k][2] = v[2]; stg[k][3] = v[3];
    }
  };
  auto store_tile = [&](int buf) {
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int row = srow + NT / CHR * (k % (NCH / 2));
      char* dst = lds + buf * BUF + (k < NCH / 2 ? row * KRS : KBUF + row * VRS) + scol;
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
  const int nt = tile1 - tile0;
  const float c = a.sm_log2;  // (not negative)
  load_tile(0);
  store_tile(0);
  __syncthreads();
  if (nt > 1) load_tile(1);
  for (int j = 0; j < nt; ++j) {
    const char* kb = lds + (NBUF == 2 ? (j & 1) * BUF : 0) + 32 * wk * KRS;
    const char* vb = lds + (NBUF == 2 ? (j & 1) * BUF : 0) + KBUF + 32 * wk * VRS;
    const int left = keys - j * KT - 32 * wk;  // the wave's keys from here on
    if (r0 < a.M && (WK == 1 || left > 0)) {
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
      if (left < 32) {  // the split's last keys: key 16 tt + 4g + i
        int lim = left - 4 * g;
        asm volatile("" : "+v"(lim));  // (keeps the compares on this branch)
#pragma unroll
        for (int tt = 0; tt < TT; ++tt)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (16 * tt + i >= lim)
#pragma unroll
              for (int qb = 0; qb < NQ; ++qb) s[tt][qb][i] = -INFINITY;
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
        for (int i = 0; i < 8; ++i) {
          const float p = __builtin_amdgcn_exp2f(fmaf(s[i / 4][qb][i % 4], c, -m_run[qb]));
          ls += p;
          bp[qb][i] = (E)p;
        }
        l_run[qb] += ls;
      }
      __builtin_amdgcn_s_setprio(1);
      const __attribute__((address_space(3))) char* vrow =
          (const __attribute__((address_space(3))) char*)vb + (4 * g + (c16 >> 2)) * VRS + (c16 & 3) * 8;
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
    if (NBUF == 1) __syncthreads();
    if (j + 1 < nt) store_tile(NBUF == 2 ? (j + 1) & 1 : 0);
    if (j + 2 < nt) load_tile(j + 2);
    __syncthreads();
  }
  float lt[NQ];
#pragma unroll
  for (int qb = 0; qb < NQ; ++qb) lt[qb] = col_sum(l_run[qb]);
  if constexpr (WK > 1) {
    // the waves' parts of the same rows: (m, l) of every wave, then O scaled to the joint maximum,
    // 16 rows at a time in the tiles' LDS, added in wave order; a wave keeps the dims of tiles wk, wk + WK ..
    __shared__ float s_ml[WK][QB][2];
    float* so = reinterpret_cast<float*>(lds);  // [waves][DT][64 lanes][4]
    static_assert(WQ * WK * DT * 1024 <= NBUF * BUF, "the waves' O fits the tiles' LDS");
    const int rr = QW * wq + c16;
#pragma unroll
    for (int qb = 0; qb < NQ; ++qb)
      if (g == 0) { s_ml[wk][16 * qb + rr][0] = m_run[qb]; s_ml[wk][16 * qb + rr][1] = lt[qb]; }
    __syncthreads();
#pragma unroll
    for (int qb = 0; qb < NQ; ++qb) {
      float m = kLowest, l = 0.f;
#pragma unroll
      for (int i = 0; i < WK; ++i) m = fmaxf(m, s_ml[i][16 * qb + rr][0]);
#pragma unroll
      for (int i = 0; i < WK; ++i) l += s_ml[i][16 * qb + rr][1] * __builtin_amdgcn_exp2f(s_ml[i][16 * qb + rr][0] - m);
      const float f = __builtin_amdgcn_exp2f(m_run[qb] - m);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<float4_t*>(so + ((w * DT + dt) * 64 + lane) * 4) = o[qb][dt] * f;
      m_run[qb] = m;
      lt[qb] = l;
      __syncthreads();
#pragma unroll
      for (int u = 0; u < (DT + WK - 1) / WK; ++u) {
        const int dt = wk + WK * u;
        if (dt >= DT) break;
        float4_t v = *reinterpret_cast<const float4_t*>(so + ((wq * DT + dt) * 64 + lane) * 4);
#pragma unroll
        for (int i = 1; i < WK; ++i) v += *reinterpret_cast<const float4_t*>(so + (((i * WQ + wq) * DT + dt) * 64 + lane) * 4);
        o[qb][u] = v;
      }
      __syncthreads();
    }
  }
  // the rows' results, or the split's partial (lane: row r0 + 16qb + c16, dims 16dt + 4g ..)
  constexpr int OT = (DT + WK - 1) / WK;
#pragma unroll
  for (int qb = 0; qb < NQ; ++qb) {
    const int r = r0 + 16 * qb + c16;
    if (r >= a.M) continue;
    const bool first = g == 0 && wk == 0;
    if (a.nsplit == 1) {
      const PrefixRow x = prefix_row(a, hk, r);
      const PrefixOwn<ET> own(a, x, m_run[qb]);
#pragma unroll
      for (int u = 0; u < OT; ++u)
        if (wk + WK * u < DT) own.write(a, x, 16 * (wk + WK * u) + 4 * g, o[qb][u], lt[qb]);
      if (a.lse && first) own.write_lse(a, x, lt[qb]);
    } else {
      const long pr = (long)sp * a.rows + (long)hk * a.M + r;
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

// The splits' partials of a row, and its own part: a work-group has 256 / D
// rows; JG groups of D / 4 threads take every JG-th split of a row, four dims a
// thread, and are added up in LDS in group order.
template <typename ET, int D>
__global__ __launch_bounds__(256) void prefix_join_kernel(PrefixArgs a) {
  constexpr int D4 = D / 4, JG = 4, RW = 256 / (D4 * JG);
  __shared__ float4_t s_o[256];
  __shared__ float2 s_ml[RW][JG];
  const int d4 = threadIdx.x % D4, grp = threadIdx.x / D4 % JG, rw = threadIdx.x / (D4 * JG);
  const long pr = (long)blockIdx.x * RW + rw;
  const bool in = pr < a.rows;
  float m = kLowest, L = 0.f;
  float4_t o = {0.f, 0.f, 0.f, 0.f};
  if (in)
    for (int s0 = grp; s0 < a.nsplit; s0 += 4 * JG) {  // four splits' loads in flight
      float2 ml[4];
      float4_t v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const long r = min(s0 + u * JG, a.nsplit - 1) * a.rows + pr;
        ml[u] = *reinterpret_cast<const float2*>(a.pml + 2 * r);
        v[u] = *reinterpret_cast<const float4_t*>(a.po + r * D + 4 * d4);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (s0 + u * JG >= a.nsplit) break;
        const float mn = fmaxf(m, ml[u].x), f = __builtin_amdgcn_exp2f(m - mn), e = __builtin_amdgcn_exp2f(ml[u].x - mn);
        o = o * f + v[u] * e;
        L = L * f + ml[u].y * e;
        m = mn;
      }
    }
  s_o[threadIdx.x] = o;
  if (d4 == 0) s_ml[rw][grp] = make_float2(m, L);
  __syncthreads();
  if (!in || grp != 0) return;
  float mm = kLowest, LL = 0.f;
  float4_t O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < JG; ++i) mm = fmaxf(mm, s_ml[rw][i].x);
#pragma unroll
  for (int i = 0; i < JG; ++i) {
    const float f = __builtin_amdgcn_exp2f(s_ml[rw][i].x - mm);
    LL += s_ml[rw][i].y * f;
    O += s_o[(rw * JG + i) * D4 + d4] * f;
  }
  const int hk = (int)pr / a.by_m;
  const PrefixRow x = prefix_row(a, hk, (int)(pr - (long)hk * a.M));
  const PrefixOwn<ET> own(a, x, mm);
  own.write(a, x, 4 * d4, O, LL);
  if (a.lse && d4 == 0) own.write_lse(a, x, LL);
}

namespace {
// How a call is cut.  At most 32 rows a kv head: the four waves of a work-group
// split a tile's keys (wq = 1, wk = 4); more: they split the rows (wq = 4, wk =
// 1).  Key splits until 768 work-groups (3 a CU) are there, each of at least 4
// tiles; up to 8 tiles one split, whose launch writes the results (4 x 8 rows on
// 1000 keys: two splits and their join 8 + 4 us).
//
// Many splits of a long prefix: work-groups of 12 waves, a CU each, whose three
// sets of waves share the rows and are joined in LDS (wk = 3): a third of the
// partials.  us a call, one set / three: 64 rows x 32 / 8 heads, D = 128, on 32768
// keys (48 splits) 72.5 / 67, 8192 35 / 30, 4096 27 / 26.5, 2048 (16 splits) 21.3 /
// 22.5; 16 rows on 32768 40 / 36, on 4096 17 / 18; D = 64, 32 / 4 heads, 64 rows on
// 4096 21.7 / 18.3, on 1500 13.4 / 14.8, 16 rows on 32768 38 / 26.
struct PrefixPlan {
  int wq, wk, nqb, nsplit;
};
PrefixPlan prefix_plan(const carekv_prefix_params& p) {
  PrefixPlan r{};
  const long M = (long)p.batch * p.seq_len * (p.n_heads / p.n_kv_heads);
  r.wq = M <= 32 ? 1 : 4;
  r.wk = M <= 32 ? 4 : 1;
  r.nqb = (int)((M + 32 * r.wq - 1) / (32 * r.wq));
  const long wgs = (long)r.nqb * p.n_kv_heads;
  auto tiles = [&]() { return ((long)p.prefix_len + 32 * r.wk - 1) / (32 * r.wk); };
  if (tiles() == 0 || wgs == 0) return r;
  auto splits = [&](long places, long least) {
    return (int)(tiles() <= 8 ? 1 : std::min(tiles(), std::max(1L, std::min(places / wgs, (tiles() + least - 1) / least))));
  };
  r.nsplit = splits(768, 4);
  if (r.wq == 4 && r.nsplit >= 12 && tiles() >= 128) {
    r.wk = 3;
    r.nsplit = splits(256, 3);
  }
  return r;
}
int check_prefix(const carekv_prefix_params* pp) {
  CAREKV_REQUIRE(pp, "null argument");
  const carekv_prefix_params& p = *pp;
  CAREKV_REQUIRE(p.head_dim == 64 || p.head_dim == 128, "head_dim must be 64 or 128");
  CAREKV_REQUIRE(p.dtype == CAREKV_F16 || p.dtype == CAREKV_BF16, "dtype must be CAREKV_F16 or CAREKV_BF16");
  CAREKV_REQUIRE(p.batch >= 0 && p.seq_len >= 0 && p.prefix_len >= 0, "negative counts");
  CAREKV_REQUIRE(p.n_heads > 0 && p.n_kv_heads > 0 && p.n_heads % p.n_kv_heads == 0,
                 "n_heads must be a positive multiple of n_kv_heads");
  CAREKV_REQUIRE(p.prefix_len < (1 << 30), "prefix_len must be below 2^30");
  CAREKV_REQUIRE((long)p.batch * p.seq_len * p.n_heads < (1L << 30), "too many rows");
  CAREKV_REQUIRE(p.prefix_len < 2 || (p.k_st >= 0 && p.v_st >= 0 && p.k_st < (1 << 22) && p.v_st < (1 << 22)),
                 "K and V row strides must be in 0 .. 2^22 elements");
  return CAREKV_OK;
}
long prefix_ws(const carekv_prefix_params& p, int ns) {
  const long rows = (long)p.batch * p.seq_len * p.n_heads;
  return ns > 1 ? ns * rows * (2 + p.head_dim) * 4 : 0;
}
}  // namespace

}  // namespace carekv

using namespace carekv;

extern "C" int64_t carekv_prefix_attn_workspace_bytes(const carekv_prefix_params* pp) {
  if (check_prefix(pp) != CAREKV_OK) return -1;
  return prefix_ws(*pp, prefix_plan(*pp).nsplit);
}

extern "C" int carekv_prefix_attn(const carekv_prefix_params* pp, const void* q, const void* k, const void* v,
                                  const void* own, const float* own_lse, void* out, float* lse, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  const int rc = check_prefix(pp);
  if (rc != CAREKV_OK) return rc;
  const carekv_prefix_params& p = *pp;
  const long rows = (long)p.batch * p.seq_len * p.n_heads;
  if (rows == 0) return CAREKV_OK;
  CAREKV_REQUIRE(q && out && (workspace || prefix_plan(p).nsplit < 2) && (p.prefix_len == 0 || (k && v)) && !own == !own_lse, "null argument");
  CAREKV_REQUIRE(!lse || lse != own_lse, "lse must not be own_lse");
  const uintptr_t bits = operand_bits(q, {{p.batch, 2 * p.q_sb}, {p.n_heads, 2 * p.q_sh}, {p.seq_len, 2 * p.q_st}}) |
                         operand_bits(k, {{p.n_kv_heads, 2 * p.k_sh}, {p.prefix_len, 2 * p.k_st}}) |
                         operand_bits(v, {{p.n_kv_heads, 2 * p.v_sh}, {p.prefix_len, 2 * p.v_st}}) |
                         (uintptr_t)workspace;
  CAREKV_REQUIRE((bits & 15) == 0, "q, k and v rows must be 16-byte aligned");
  const PrefixPlan plan = prefix_plan(p);
  const int ns = plan.nsplit;
  if (workspace_bytes < prefix_ws(p, ns)) {
    set_error("carekv_prefix_attn: workspace too small (%lld < %lld)", (long long)workspace_bytes,
              (long long)prefix_ws(p, ns));
    return CAREKV_ESPACE;
  }
  PrefixArgs a{};
  a.q = (const char*)q; a.k = (const char*)k; a.v = (const char*)v; a.own = (const char*)own; a.own_lse = own_lse;
  a.out = (char*)out; a.lse = lse;
  a.q_sb = 2 * p.q_sb; a.q_sh = 2 * p.q_sh; a.q_st = 2 * p.q_st; a.k_sh = 2 * p.k_sh; a.k_st = 2 * p.k_st;
  a.v_sh = 2 * p.v_sh; a.v_st = 2 * p.v_st; a.o_sb = 2 * p.out_sb; a.o_sh = 2 * p.out_sh; a.o_st = 2 * p.out_st;
  a.w_sb = 2 * p.own_sb; a.w_sh = 2 * p.own_sh; a.w_st = 2 * p.own_st;
  a.B = p.batch; a.Hq = p.n_heads; a.Hkv = p.n_kv_heads; a.G = p.n_heads / p.n_kv_heads; a.T = p.seq_len;
  a.P = p.prefix_len; a.M = p.batch * a.G * p.seq_len; a.rows = rows; a.nqb = plan.nqb; a.nsplit = ns;
  a.by_t = FastDiv(a.T); a.by_g = FastDiv(a.G); a.by_m = FastDiv(a.M);
  a.by_nqb = FastDiv(std::max(a.nqb, 1)); a.by_nsplit = FastDiv(std::max(ns, 1));
  a.po = (float*)workspace;
  a.pml = a.po + ns * rows * p.head_dim;
  a.sm_log2 = (float)(std::fabs((double)p.sm_scale) * 1.4426950408889634074);
  a.q_sign = p.sm_scale < 0.f ? 0x80008000u : 0u;
  a.q_keep = a.sm_log2 == 0.f ? 0u : ~0u;
  if (a.sm_log2 == 0.f) a.sm_log2 = 1.f;
  uintptr_t rows8 = operand_bits(out, {{p.batch, a.o_sb}, {p.n_heads, a.o_sh}, {p.seq_len, a.o_st}});
  if (own) rows8 |= operand_bits(own, {{p.batch, a.w_sb}, {p.n_heads, a.w_sh}, {p.seq_len, a.w_st}});
  a.al8 = (rows8 & 7) == 0;
  hipStream_t s = (hipStream_t)stream;
  const long wgs = (long)a.nqb * a.Hkv * ns;
  CAREKV_REQUIRE(grid_fits(wgs, 768) && (ns == 1 || grid_fits(rows / (256 / p.head_dim) + 1, 256)), "too many rows");
  return dispatch_elem_d(p.dtype, p.head_dim, [&](auto et, auto d) {
    using ET = decltype(et);
    constexpr int D = decltype(d)::value;
    if (ns > 0) {
      const dim3 grid((unsigned)wgs), block(64 * plan.wq * plan.wk);
      if (plan.wq == 1) hipLaunchKernelGGL((prefix_attn_kernel<ET, D, 1, 4>), grid, block, 0, s, a);
      else if (plan.wk == 1) hipLaunchKernelGGL((prefix_attn_kernel<ET, D, 4, 1>), grid, block, 0, s, a);
      else hipLaunchKernelGGL((prefix_attn_kernel<ET, D, 4, 3>), grid, block, 0, s, a);
      CAREKV_CHECK_LAUNCH("prefix_attn");
    }
    if (ns != 1) {
      constexpr int RW = 256 / D;
      hipLaunchKernelGGL((prefix_join_kernel<ET, D>), dim3((unsigned)((rows + RW - 1) / RW)), dim3(256), 0, s, a);
      CAREKV_CHECK_LAUNCH("prefix_join");
    }
    return CAREKV_OK;
  });
}
