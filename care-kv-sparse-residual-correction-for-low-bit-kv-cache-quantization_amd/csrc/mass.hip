// Attention weight that each key has gathered (attention_mass):
//   mass[b][g][j] = sum over the query heads h of kv head g and the query rows
//   i that see key j of e^(scale q_i . k_j - lse_i)
// with lse_i the log-sum-exp of row i's visible scores, given or computed here.
// Query row i stands at position q_start + i and sees the keys j below
// min(length, position + 1) (not causal: below the length); rows from q_length
// on (the padding of a ragged batch) see nothing.
//
// mass_kernel, key-stationary: a work-group keeps 256 keys (8 waves of 32, the
// A operand of S^T = K Q^T in registers) and walks over 64-row tiles of q
// staged in LDS, so that a key's weights add up in registers and nothing of
// size queries x keys is written.  Heads are walked one after the other, each
// from the first row that sees the block; heads of fewer than 32 rows as one
// list.  A work-group takes a pair of blocks, early and late, whose causal walks
// have the same length together, or an equal part of a pair's walk; the parts'
// sums are added in order by mass_sum_kernel.
//
// stats_kernel, its mirror image for calls without lse: 256 query rows
// stationary, key tiles walked, each lane with its own (reference, sum) per row.
// The reference is no maximum, only a value that no logit passes by 2^64: sums
// stay in 32-bit range, their accuracy is relative, so that it need not move
// with every larger score.  mass_join_kernel joins the walks' parts; those of few
// rows are joined by the mass walks.
//
// mass_few_kernel, at most 16 rows a kv head (a decode step): a work-group a
// (sequence, kv head), the scores of all keys in LDS, K read once, one launch.
// Past kFewBytes of K a head the keys are cut into parts (mass_scores_kernel: K
// read once, the scores to memory; mass_weigh_kernel: their weights), up to 2048
// work-groups.  The limit is that of an eager call, where the second launch and
// the workspace cost 4 us of host time: 8 heads, D = 128, 4 rows on 1280 keys (320
// KB) 13.8 us in one launch, 15.7 in two whatever the keys up to 4096.  In a graph
// it depends on the heads too, one launch / two: 8 heads, D = 128, 4 rows on 512
// keys (128 KB) 8.3 / 7.8, 1024 11.5 / 8.0, 2048 18.9 / 8.4, 4096 33.7 / 8.4; 128
// heads, D = 64, 8 rows on 2303 keys (288 KB) 14.9 / 16.4, 4000 22.0 / 21.2: few
// heads lose up to 5 us there below the limit.  Decode steps on 8 x 8192
// keys, 32 / 8 heads (134 MB) 27 us, on 16 x 6000, 32 / 32 heads (786 MB) 160, 4.9
// TB/s (as walks 64 and 374).
//
// Measured, D = 128, 8192 causal rows with lse: 32 / 8 heads 324 us + 5 for the
// sum of the parts (275 GFLOP of visible products, 1.07e9 exponentials: 0.84
// PFLOP/s; in bursts after a pause 340-360), 32 / 32 heads 318, without lse 32 / 8
// heads 632; long uncut walks reach 1.0 PFLOP/s.  Bound: a 16 x 16 x 32 product
// with the exponential and two fused multiply-adds of its four scores a lane takes
// a SIMD 25 cycles at best (measured in registers alone; the product itself 16),
// 180 us of the 324.  Against 321 then: blocks in order instead of pairs, 2048
// work-groups, 350; LDS rows padded by 16 bytes (9.0 cycles a read against 5.6)
// 360; masked wave tiles not skipped 337.  Before these, against 355-370: 4 waves
// of 64 keys 363, 32 x 32 products 374; not measured since.  A window of 64 rows
// on 4 x 8191 keys: 29 us statistics, 31 us weights, 8 us each before the first
// products and 1.1 us a tile and CU, which two work-groups a CU (or two tiles on
// their way) change by little: K (67 MB) is not what bounds them.
//
// Sums: a lane adds at most kFlush tiles' weights before they go to an outer
// sum, so that a key's total over 2^15 rows keeps the accuracy of a short sum.
// A row's statistics are (M, w): a weight is 2^(x - M) w, with w = 1 / sum, or
// for a given lse the part of lse log2(e) that a 32-bit M does not hold.
#include <algorithm>

#include "fast_div.h"
#include "mfma16.h"

namespace carekv {

struct MassArgs {
  const char* q;
  const char* k;
  const float* lse;        // [B][Hq][Tq], or null
  const int32_t* q_start;  // [B], or null: the rows are the last of the length
  const int32_t* lengths;  // [B], or null
  const int32_t* q_lengths;  // [B], or null
  float* out;
  float* part;             // [B][Hkv][rows][nsk][2] reference (base 2), sum
  float* stat;             // [B][Hkv][rows][2] M, w (no lse)
  float* opart;            // [parts][B][Hkv][Tk], parts > 1
  long q_sb, q_sh, q_st, k_sb, k_sh, k_st;  // bytes
  long o_sb, o_sh;                          // elements
  int B, Hq, Hkv, G, Tq, Tk, causal, accumulate;
  int nkb, parts;          // mass walks: key blocks, parts that a pair of blocks' walk is cut into
  int nqb, nsk;            // statistics: row blocks, parts of a walk
  int fold;                // mass_kernel joins the parts of its rows' statistics itself
  FastDiv by_nhb, by_hkv, by_tq, by_kpairs, by_qpairs, by_parts, by_nsk;  // nhb = B Hkv, pairs of blocks
  int nseg, seg;           // a mass walk: nseg lists of seg rows
  float sm_log2;
};

constexpr int kMassKeys = 256, kMassTile = 64, kFlush = 8, kFewRows = 16, kFewLds = 131072, kFewBytes = 320 << 10, kFoldRows = 256;

// A sequence's visible keys: row t < nq sees j < min(len, qs + t + 1), not causal: j < len.
struct MassSeq {
  int len, nq;
  long qs;
};
__device__ __forceinline__ MassSeq mass_seq(const MassArgs& a, int b) {
  MassSeq s;
  s.len = a.lengths ? min(max(a.lengths[b], 0), a.Tk) : a.Tk;
  s.nq = a.q_lengths ? min(max(a.q_lengths[b], 0), a.Tq) : a.Tq;
  s.qs = a.q_start ? (long)a.q_start[b] : (long)s.len - s.nq;
  return s;
}
__device__ __forceinline__ int mass_limit(const MassArgs& a, const MassSeq& s, int t) {
  return t >= s.nq ? 0 : a.causal ? (int)max(0L, min((long)s.len, s.qs + t + 1)) : s.len;
}

// (M, w) of a row with log-sum-exp l: l log2(e) = M + rest, M the rounded
// product, rest what it lost.  Infinite l: (inf, 0), whose row is masked (0 times what it holds may be NaN).  NaN
// goes on as NaN.
__device__ __forceinline__ float2 lse_stat(float l) {
  float2 st = make_float2(INFINITY, 0.f);
  if (!(fabsf(l) >= 1e30f)) {
    st.x = l * kLog2e;
    const float rest = fmaf(l, kLog2e, -st.x) + l * 1.9259629911266174e-8f;  // log2(e) - float(log2(e))
    st.y = __builtin_amdgcn_exp2f(-rest);
  }
  return st;
}

template <typename V8>
__device__ __forceinline__ V8 load8(const char* p) {
  V8 x;
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  __builtin_memcpy(&x, &v, 16);
  return x;
}

// (M, w) of a row, given to the first of its N lanes (u = 0 .. N - 1), from the parts of its walk, eight of a lane's
// loads in flight.  A row that sees nothing has (inf, 0): weights of 0.
template <int N>
__device__ __forceinline__ float2 join_parts(const float2* p, int nsk, int u) {
  float mx = kLowest, l = 0.f;
  for (int s0 = u; s0 < nsk; s0 += 8 * N) {
    float2 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = p[min(s0 + N * i, nsk - 1)];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (s0 + N * i >= nsk) break;
      const float m = fmaxf(mx, v[i].x);
      l = l * __builtin_amdgcn_exp2f(mx - m) + v[i].y * __builtin_amdgcn_exp2f(v[i].x - m);
      mx = m;
    }
  }
#pragma unroll
  for (int o = 1; o < N; o <<= 1) {
    const float m = fmaxf(mx, __shfl_xor(mx, o, 64)), f = l * __builtin_amdgcn_exp2f(mx - m);
    l = f + __shfl_xor(f, o, 64);
    mx = m;
  }
  return l != 0.f ? make_float2(mx, 1.f / l) : make_float2(INFINITY, 0.f);
}

// GIVEN: with the rows' log-sum-exp.
template <typename ET, int D, bool GIVEN>
__global__ __launch_bounds__(512, 4) void mass_kernel(MassArgs a) {
  using V8 = typename ET::V8;
  constexpr int TT = kMassKeys / 128, QT = kMassTile, KS = D / 32, QRS = 2 * D + 32, CHR = D / 8, NCH = QT * CHR / 512;
  __shared__ __align__(16) char lds[2][QT * QRS];
  static_assert(QT == 64, "a wave has a tile's rows");
  __shared__ float2 s_st[2][QT];
  __shared__ int s_lim[2][QT];
  __shared__ int s_off[8];  // a wave's share of the rows has one of infinite lse
  __shared__ float2 s_row[kFoldRows];  // every row's (M, w), where the statistics' parts are joined here
  __shared__ float s_sum[4 * TT][512];  // the outer sums: the registers they would take spill others
  // Sequences and heads go round the XCDs, the blocks of one part run together: they meet in one L2.
  const int nhb = a.by_nhb.d, rest = (int)blockIdx.x / a.by_nhb, hb = blockIdx.x - rest * nhb;
  const int pt = rest / a.by_kpairs, pair = rest - pt * a.by_kpairs.d;
  const int b = hb / a.by_hkv, hk = hb - b * a.Hkv;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c16 = lane & 15;
  if (!GIVEN && a.fold) {  // (256 rows, two lanes each; before the length is known)
    const int r = threadIdx.x / 2, rows = a.G * a.Tq;
    const float2 st = join_parts<2>(reinterpret_cast<const float2*>(a.part) + ((long)hb * rows + min(r, rows - 1)) * a.nsk,
                                    a.nsk, threadIdx.x & 1);
    if (threadIdx.x % 2 == 0) s_row[r] = st;
    __syncthreads();
  }
  const MassSeq sq = mass_seq(a, b);
  const long hrow = (long)hb * a.G * a.Tq;  // first row of this (sequence, kv head) in stat / lse
  const bool listed = a.nseg > 1 || a.G == 1;  // a list is a head's rows
  // Rows of infinite lse are masked, whatever they hold: where there are any, every tile looks for them.  (Found here,
  // 1 % of a prompt's walks; a flag of each tile's rows, read before its first branch, cost 4 %.)
  bool off = false;
  if (GIVEN && listed)
    for (int r0 = threadIdx.x; r0 < a.G * a.Tq; r0 += 512 * 8) {
      float l[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) l[i] = a.lse[hrow + min(r0 + 512 * i, a.G * a.Tq - 1)];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (fabsf(l[i]) >= 1e30f) off |= min(r0 + 512 * i, a.G * a.Tq - 1) % a.by_tq < sq.nq;
    }
  if (GIVEN) {
    off = __any(off);
    if (lane == 0) s_off[w] = off;
  }
  const int seg = listed ? sq.nq : a.seg;  // rows of a list
  // those below first_row see nothing of block kb
  auto first_row = [&](int kb) {
    if (kb * kMassKeys >= sq.len) return seg;
    return a.causal && listed ? (int)min((long)seg, max(0L, (long)kb * kMassKeys - sq.qs)) : 0;
  };
  auto tiles_of = [&](int kb) { return (seg - first_row(kb) + QT - 1) / QT * a.nseg; };
  // The pair's walks, one after the other, as one: this part's tiles of it.
  const int kb_b = a.nkb - 1 - pair, n_a = tiles_of(pair), n_all = n_a + (kb_b > pair ? tiles_of(kb_b) : 0);
  const int lo = part_start(n_all, pt, a.by_parts), hi = part_start(n_all, pt + 1, a.by_parts);
  float* dst = a.parts > 1 ? a.opart + ((long)pt * nhb + hb) * a.Tk : a.out + b * a.o_sb + hk * a.o_sh;
  const uint32_t off0 = (uint32_t)(threadIdx.x / CHR * a.q_st + (threadIdx.x % CHR) * 16);
  const char* qbase = a.q + b * a.q_sb + (long)hk * a.G * a.q_sh;
#pragma unroll 1
  for (int f = 0; f < (kb_b > pair ? 2 : 1); ++f) {
  const int kb = f ? kb_b : pair, j0 = kb * kMassKeys + 16 * TT * w;  // the block, the wave's first key
  const int t_first = first_row(kb), t_end = seg, per = max(1, (t_end - t_first + QT - 1) / QT);
  const int at = max(lo - (f ? n_a : 0), 0), nt = min(hi, f ? n_all : n_a) - (f ? n_a : 0) - at;
  int sg = 0, i0 = at;  // the tile loaded next: list, first row
  while (i0 >= per) { i0 -= per; ++sg; }  // (at most nseg turns)
  i0 = t_first + i0 * QT;
  // K operands: tokens j0 + 16 tt + c16, dims 32 s + 8 g .. (keys past the end: the last one, masked below)
  V8 kf[TT][KS];
  if (nt > 0) {
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) {
      const char* kp = a.k + b * a.k_sb + hk * a.k_sh + (long)min(j0 + 16 * tt + c16, a.Tk - 1) * a.k_st;
#pragma unroll
      for (int s = 0; s < KS; ++s) kf[tt][s] = load8<V8>(kp + (32 * s + 8 * g) * 2);
    }
  }
  uint32_t stg[NCH][4];
  float2 n_st = make_float2(0.f, 0.f);
  int n_lim = 0, turn = 0, sturn = 0;  // the wave of the tile loaded / stored next
  // A list's rows lie one row stride apart: a tile is a buffer resource of its rows (those behind the list's
  // end read as zeros), a thread's offsets in it stay the same.  Other lists find their rows one by one.
  auto load_tile = [&]() {
    if (listed) {
      const __amdgpu_buffer_rsrc_t rq = make_rsrc(qbase + sg * a.q_sh + i0 * a.q_st,
                                                  (uint32_t)((min(QT, t_end - i0) - 1) * a.q_st + 2 * D));
#pragma unroll
      for (int k = 0; k < NCH; ++k) {
        uint32_t off = off0;
        asm volatile("" : "+v"(off));  // (added here, not kept in a register of its own)
        const auto v = __builtin_amdgcn_raw_buffer_load_b128(rq, off + (uint32_t)(512 / CHR * k * a.q_st), 0, 0);
        stg[k][0] = v[0]; stg[k][1] = v[1]; stg[k][2] = v[2]; stg[k][3] = v[3];
      }
    } else {
#pragma unroll
      for (int k = 0; k < NCH; ++k) {
        const int i = i0 + (int)threadIdx.x / CHR + 512 / CHR * k, h = i / a.by_tq, t = i - h * a.Tq;
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (i < t_end)
          v = *reinterpret_cast<const uint4*>(qbase + h * a.q_sh + t * a.q_st + (threadIdx.x % CHR) * 16);
        stg[k][0] = v.x; stg[k][1] = v.y; stg[k][2] = v.z; stg[k][3] = v.w;
      }
    }
    // the rows' statistics, by another wave every tile, as they lie: they are turned into (M, w) when they are
    // stored, so that no wave waits for them here
    if (w == turn) {
      const int i = i0 + lane;
      int h = sg, t = i;
      if (!listed) {
        h = i / a.by_tq;
        t = i - h * a.Tq;
        n_lim = i < t_end ? mass_limit(a, sq, t) : 0;
      }
      const long r = hrow + (long)h * a.Tq + t;
      n_st = make_float2(INFINITY, 0.f);
      if (i < t_end) {
        if (GIVEN) n_st.x = a.lse[r];
        else if (a.fold) n_st = s_row[h * a.Tq + t];
        else n_st = *reinterpret_cast<const float2*>(a.stat + 2 * r);
      }
    }
    turn = (turn + 1) & 7;
    i0 += QT;
    if (i0 >= t_end) { i0 = t_first; ++sg; }
  };
  auto store_tile = [&](int buf) {
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int row = threadIdx.x / CHR + 512 / CHR * k;
      *reinterpret_cast<uint4*>(lds[buf] + row * QRS + (threadIdx.x % CHR) * 16) =
          make_uint4(stg[k][0], stg[k][1], stg[k][2], stg[k][3]);
    }
    if (w == sturn) {
      if (!listed) s_lim[buf][lane] = n_lim;
      s_st[buf][lane] = a.lse ? lse_stat(n_st.x) : n_st;  // (with GIVEN the form without lse spills four registers)
    }
    sturn = (sturn + 1) & 7;
  };
  float acc[4 * TT];
#pragma unroll
  for (int i = 0; i < 4 * TT; ++i) { acc[i] = 0.f; s_sum[i][threadIdx.x] = 0.f; }
  int ci = i0;  // first row of the tile computed next
  if (nt > 0) {
    load_tile();
    store_tile(0);
  }
  __syncthreads();
  const int care = GIVEN ? __builtin_amdgcn_readfirstlane(__any(s_off[lane & 7] != 0)) : 0;
  int ni = i0;
  if (nt > 1) load_tile();
  for (int j = 0; j < nt; ++j) {
    const int buf = j & 1;
    // (a wave whose keys no row of the tile sees has nothing to add)
    if (!(listed && (j0 >= sq.len || (a.causal && sq.qs + min(ci + QT, t_end) - 1 < j0)))) {
    // some pair of the tile and the wave's keys is masked
    const bool edge = !listed || ci + QT > t_end || j0 + 16 * TT > sq.len ||
                      (a.causal && sq.qs + ci + 1 < j0 + 16 * TT) || care != 0;
    // the next 16 rows' products are issued before this one's exponentials: they run side by side
    float4_t s[2][TT];
    auto scores = [&](int qb, float4_t* x) {
#pragma unroll
      for (int tt = 0; tt < TT; ++tt) x[tt] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const V8 qf = load8<V8>(lds[buf] + (16 * qb + c16) * QRS + (32 * ks + 8 * g) * 2);
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) x[tt] = ET::mfma(kf[tt][ks], qf, x[tt]);
      }
    };
    scores(0, s[0]);
    if (!edge) {
#pragma unroll
      for (int qb = 0; qb < QT / 16; ++qb) {
        if (qb + 1 < QT / 16) scores(qb + 1, s[(qb + 1) & 1]);
        const float2 st = s_st[buf][16 * qb + c16];
#pragma unroll
        for (int i = 0; i < 4 * TT; ++i)
          acc[i] = fmaf(__builtin_amdgcn_exp2f(fmaf(s[qb & 1][i / 4][i % 4], a.sm_log2, -st.x)), st.y, acc[i]);
      }
    } else {
#pragma unroll
      for (int qb = 0; qb < QT / 16; ++qb) {
        if (qb + 1 < QT / 16) scores(qb + 1, s[(qb + 1) & 1]);
        const float2 st = s_st[buf][16 * qb + c16];
        const int i0c = ci + 16 * qb + c16;
        const int see = GIVEN && st.y == 0.f ? 0 : !listed ? s_lim[buf][16 * qb + c16] : i0c < t_end ? mass_limit(a, sq, i0c) : 0;
        const int lim = see - j0 - 4 * g;  // token 16 tt + i of the lane is seen below it
#pragma unroll
        for (int i = 0; i < 4 * TT; ++i) {
          const float p = __builtin_amdgcn_exp2f(fmaf(s[qb & 1][i / 4][i % 4], a.sm_log2, -st.x));
          acc[i] = 16 * (i / 4) + i % 4 < lim ? fmaf(p, st.y, acc[i]) : acc[i];
        }
      }
    }
    }
    if ((j + 1) % kFlush == 0) {
#pragma unroll
      for (int i = 0; i < 4 * TT; ++i) { s_sum[i][threadIdx.x] += acc[i]; acc[i] = 0.f; }
    }
    ci = ni;
    if (j + 1 < nt) store_tile((j + 1) & 1);
    if (j + 2 < nt) { ni = i0; load_tile(); }
    __syncthreads();
  }
  // over the 16 query columns, in a fixed order
#pragma unroll
  for (int i = 0; i < 4 * TT; ++i) {
    float v = s_sum[i][threadIdx.x] + acc[i];
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) v += __shfl_xor(v, o, 64);
    const int key = j0 + 16 * (i / 4) + 4 * g + i % 4;
    if (c16 == 0 && key < a.Tk) dst[key] = a.accumulate && a.parts == 1 ? dst[key] + v : v;
  }
  }
}

// The parts of the walks, in order.
__global__ __launch_bounds__(256) void mass_sum_kernel(MassArgs a) {
  const long n = (long)a.B * a.Hkv * a.Tk, i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float v = 0.f;
  for (int p = 0; p < a.parts; ++p) v += a.opart[p * n + i];
  const long hb = (uint32_t)i / (uint32_t)a.Tk, b = (int)hb / a.by_hkv;
  float* dst = a.out + b * a.o_sb + (hb - b * a.Hkv) * a.o_sh + (i - hb * a.Tk);
  *dst = a.accumulate ? *dst + v : v;
}

template <typename ET, int D>
__global__ __launch_bounds__(512, 4) void stats_kernel(MassArgs a) {
  using V8 = typename ET::V8;
  constexpr int TT = 2, KT = kMassTile, KS = D / 32, KRS = 2 * D + 32, CHR = D / 8, NCH = KT * CHR / 512;
  constexpr float kOver = 64.f;
  __shared__ __align__(16) char lds[2][KT * KRS];
  const int rest = (int)blockIdx.x / a.by_nhb, hb = blockIdx.x - rest * a.by_nhb.d;
  const int sp = rest / a.by_qpairs, pair = rest - sp * a.by_qpairs.d;
  const int b = hb / a.by_hkv, hk = hb - b * a.Hkv;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c16 = lane & 15;
  const int rows = a.G * a.Tq;
  const MassSeq sq = mass_seq(a, b);
  uint32_t off[NCH];
#pragma unroll
  for (int k = 0; k < NCH; ++k)
    off[k] = (uint32_t)((threadIdx.x / CHR + 512 / CHR * k) * a.k_st + (threadIdx.x % CHR) * 16);
  const char* kbase = a.k + b * a.k_sb + hk * a.k_sh;
  // tiles of the keys that some row of block qb sees: its rows' furthest limit, a head's last row below nq where it
  // has one
  auto tiles_of = [&](int qb) {
    const int ra = qb * 256, rz = min(ra + 256, rows) - 1;
    const int hz = rz / a.by_tq, ta = ra - hz * a.Tq, t = min(ta < 0 ? a.Tq - 1 : rz - hz * a.Tq, sq.nq - 1);
    return t < max(ta, 0) ? 0 : (mass_limit(a, sq, t) + KT - 1) / KT;
  };
  // The pair's walks, one after the other, as one: this part's tiles of it.
  const int qb_b = a.nqb - 1 - pair, n_a = tiles_of(pair), n_all = n_a + (qb_b > pair ? tiles_of(qb_b) : 0);
  const int from = part_start(n_all, sp, a.by_nsk), to = part_start(n_all, sp + 1, a.by_nsk);
#pragma unroll 1
  for (int f = 0; f < (qb_b > pair ? 2 : 1); ++f) {
  const int r0 = (f ? qb_b : pair) * 256 + 16 * TT * w;
  const int t0 = max(from - (f ? n_a : 0), 0), nt = min(to, f ? n_all : n_a) - (f ? n_a : 0) - t0;
  V8 qf[TT][KS];
  int lim[4 * TT], lo = 0x7fffffff;
#pragma unroll
  for (int tt = 0; tt < TT; ++tt) {
    const int r = min(r0 + 16 * tt + c16, rows - 1), h = r / a.by_tq, t = r - h * a.Tq;
    const char* qp = a.q + b * a.q_sb + ((long)hk * a.G + h) * a.q_sh + (long)t * a.q_st;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[tt][s] = load8<V8>(qp + (32 * s + 8 * g) * 2);
  }
  // keys that the lane's rows r0 + 16 tt + 4 g + i see, and the furthest and nearest end over the work-group / wave
  int hi = 0;
#pragma unroll
  for (int tt = 0; tt < TT; ++tt) {
    int r = r0 + 16 * tt + 4 * g, t = r % a.by_tq;
#pragma unroll
    for (int i = 0; i < 4; ++i, ++r) {
      lim[4 * tt + i] = r < rows ? mass_limit(a, sq, t) : 0;
      t = t + 1 == a.Tq ? 0 : t + 1;
      lo = min(lo, lim[4 * tt + i]);
      hi = max(hi, lim[4 * tt + i]);
    }
  }
#pragma unroll
  for (int o = 16; o < 64; o <<= 1) {
    lo = min(lo, __shfl_xor(lo, o, 64));
    hi = max(hi, __shfl_xor(hi, o, 64));
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  uint32_t stg[NCH][4];
  auto load_tile = [&](int j) {  // (keys behind the sequence's end read as zeros; they are masked)
    const int k0 = (t0 + j) * KT;
    const __amdgpu_buffer_rsrc_t rk = make_rsrc(kbase + k0 * a.k_st, (uint32_t)((min(KT, sq.len - k0) - 1) * a.k_st + 2 * D));
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const auto v = __builtin_amdgcn_raw_buffer_load_b128(rk, off[k], 0, 0);
      stg[k][0] = v[0]; stg[k][1] = v[1]; stg[k][2] = v[2]; stg[k][3] = v[3];
    }
  };
  auto store_tile = [&](int buf) {
#pragma unroll
    for (int k = 0; k < NCH; ++k)
      *reinterpret_cast<uint4*>(lds[buf] + (threadIdx.x / CHR + 512 / CHR * k) * KRS + (threadIdx.x % CHR) * 16) =
          make_uint4(stg[k][0], stg[k][1], stg[k][2], stg[k][3]);
  };
  float m[4 * TT], l[4 * TT];
#pragma unroll
  for (int i = 0; i < 4 * TT; ++i) { m[i] = kLowest; l[i] = 0.f; }
  if (nt > 0) {
    load_tile(0);
    store_tile(0);
  }
  __syncthreads();
  if (nt > 1) load_tile(1);
  for (int j = 0; j < nt; ++j) {
    const int buf = j & 1, k0 = (t0 + j) * KT;
    if (k0 < hi) {
      const bool edge = k0 + KT > lo;
      float4_t sb[2][TT];
      auto scores = [&](int kb, float4_t* y) {
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) y[tt] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const V8 kf = load8<V8>(lds[buf] + (16 * kb + c16) * KRS + (32 * ks + 8 * g) * 2);
#pragma unroll
          for (int tt = 0; tt < TT; ++tt) y[tt] = ET::mfma(qf[tt][ks], kf, y[tt]);
        }
      };
      scores(0, sb[0]);
#pragma unroll
      for (int kb = 0; kb < KT / 16; ++kb) {
        if (kb + 1 < KT / 16) scores(kb + 1, sb[(kb + 1) & 1]);
        const float4_t* s = sb[kb & 1];
        float x[4 * TT], top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4 * TT; ++i) x[i] = fmaf(s[i / 4][i % 4], a.sm_log2, -m[i]);
        if (edge) {
          const int key = k0 + 16 * kb + c16;
#pragma unroll
          for (int i = 0; i < 4 * TT; ++i)
            if (key >= lim[i]) x[i] = -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < 4 * TT; i += 2) top = fmaxf(fmaxf(top, x[i]), x[i + 1]);
        if (__any(top > kOver)) {  // some lane's logit is past its reference by 2^64: it becomes the reference
#pragma unroll
          for (int i = 0; i < 4 * TT; ++i) {
            if (x[i] > kOver) {
              const float mn = s[i / 4][i % 4] * a.sm_log2;
              l[i] *= __builtin_amdgcn_exp2f(m[i] - mn);
              m[i] = mn;
              x[i] = fmaf(s[i / 4][i % 4], a.sm_log2, -mn);  // (what the product's rounding left)
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 4 * TT; ++i) l[i] += __builtin_amdgcn_exp2f(x[i]);
      }
    }
    if (j + 1 < nt) store_tile((j + 1) & 1);
    if (j + 2 < nt) load_tile(j + 2);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4 * TT; ++i) {
    float mm = m[i];
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) mm = fmaxf(mm, __shfl_xor(mm, o, 64));
    float v = l[i] * __builtin_amdgcn_exp2f(m[i] - mm);
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) v += __shfl_xor(v, o, 64);
    const int r = r0 + 16 * (i / 4) + 4 * g + i % 4;
    if (c16 == 0 && r < rows) {
      float* p = a.part + 2 * (((long)hb * rows + r) * a.nsk + sp);
      p[0] = mm;
      p[1] = v;
    }
  }
  }
}

// (M, w) of every row from the parts of its walk.
__global__ __launch_bounds__(256) void mass_join_kernel(MassArgs a) {
  const long i = ((long)blockIdx.x * 256 + threadIdx.x) / 8;  // 8 lanes a row
  const bool in = i < (long)a.B * a.Hq * a.Tq;
  const float2 st = join_parts<8>(reinterpret_cast<const float2*>(a.part) + (in ? i : 0) * a.nsk, a.nsk, threadIdx.x & 7);
  if (in && threadIdx.x % 8 == 0) reinterpret_cast<float2*>(a.stat)[i] = st;
}

// At most 16 rows a kv head: 16 waves take 64 keys each in turn.  Lane: keys
// 16 tt + 4 g + i, row c16.
template <typename ET, int D>
__global__ __launch_bounds__(1024) void mass_few_kernel(MassArgs a, int stride) {
  using V8 = typename ET::V8;
  constexpr int KS = D / 32, TT = 4;
  __shared__ __align__(16) float sc[kFewLds / 4];  // [rows][stride] base-2 logits
  __shared__ float s_m[16][16], s_l[16][16];
  __shared__ float2 s_st[16];
  const int hb = blockIdx.x, b = hb / a.by_hkv, hk = hb - b * a.Hkv, rows = a.G * a.Tq;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c16 = lane & 15;
  const int r = min(c16, rows - 1), h = r / a.by_tq, t = r - h * a.Tq;
  V8 qf[KS];
  const char* qp = a.q + b * a.q_sb + ((long)hk * a.G + h) * a.q_sh + (long)t * a.q_st;
#pragma unroll
  for (int s = 0; s < KS; ++s) qf[s] = load8<V8>(qp + (32 * s + 8 * g) * 2);
  const char* kbase = a.k + b * a.k_sb + hk * a.k_sh;
  V8 kf[TT][KS];
  auto load_keys = [&](int j) {  // (keys behind the sequence are masked, whatever they hold)
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) {
      const char* kp = kbase + (long)min(16 * (TT * j + tt) + c16, a.Tk - 1) * a.k_st;
#pragma unroll
      for (int s = 0; s < KS; ++s) kf[tt][s] = load8<V8>(kp + (32 * s + 8 * g) * 2);
    }
  };
  load_keys(w);  // on their way before the length is known
  const MassSeq sq = mass_seq(a, b);
  const int lim = c16 < rows ? mass_limit(a, sq, t) : 0;
  const int nt = (sq.len + 16 * TT - 1) / (16 * TT);  // turns with keys
  float m = kLowest, l = 0.f;
  for (int j = w; j < nt; j += 16) {
    float4_t s[TT];
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) s[tt] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int tt = 0; tt < TT; ++tt) s[tt] = ET::mfma(kf[tt][ks], qf[ks], s[tt]);
    if (j + 16 < nt) load_keys(j + 16);
    float mx = m;
#pragma unroll
    for (int i = 0; i < 4 * TT; ++i) {
      const int key = 16 * (TT * j + i / 4) + 4 * g + i % 4;
      const float x = s[i / 4][i % 4] * a.sm_log2;
      s[i / 4][i % 4] = key < lim ? x : -INFINITY;
      mx = fmaxf(mx, s[i / 4][i % 4]);
    }
    l *= __builtin_amdgcn_exp2f(m - mx);
    m = mx;
#pragma unroll
    for (int i = 0; i < 4 * TT; ++i) l += __builtin_amdgcn_exp2f(s[i / 4][i % 4] - m);
    if (c16 < rows) {
#pragma unroll
      for (int tt = 0; tt < TT; ++tt) *reinterpret_cast<float4_t*>(sc + c16 * stride + 16 * (TT * j + tt) + 4 * g) = s[tt];
    }
  }
  const float mw = col_max(m), lw = col_sum(l * __builtin_amdgcn_exp2f(m - mw));
  if (g == 0) { s_m[w][c16] = mw; s_l[w][c16] = lw; }
  __syncthreads();
  if (threadIdx.x < 16) {
    float2 st = make_float2(INFINITY, 0.f);
    if ((int)threadIdx.x < rows) {
      if (a.lse) {
        st = lse_stat(a.lse[(long)hb * rows + threadIdx.x]);
      } else {
        float mx = kLowest, ls = 0.f;
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s_m[i][threadIdx.x]);
        for (int i = 0; i < 16; ++i) ls += s_l[i][threadIdx.x] * __builtin_amdgcn_exp2f(s_m[i][threadIdx.x] - mx);
        if (ls != 0.f) st = make_float2(mx, 1.f / ls);
      }
    }
    s_st[threadIdx.x] = st;
  }
  __syncthreads();
  float* dst = a.out + b * a.o_sb + hk * a.o_sh;
  for (int key = threadIdx.x; key < a.Tk; key += 1024) {
    float v = 0.f;
    if (key < sq.len)
      for (int i = 0; i < rows; ++i) {
        const float x = sc[i * stride + key];
        const float2 st = s_st[i];
        // (masked: -inf; NaN goes on, but not from a row of infinite lse)
        if (x != -INFINITY && st.y != 0.f) v = fmaf(__builtin_amdgcn_exp2f(x - st.x), st.y, v);
      }
    dst[key] = a.accumulate ? dst[key] + v : v;
  }
}

// At most 16 rows a kv head on more keys than a work-group should read alone: the keys are cut into parts, a
// work-group (4 waves of 64 keys in turn) each.  Its base-2 logits go to `sc` [B Hkv][rows][stride] (masked: -inf),
// every row's (reference, sum) to part [B Hkv][rows][nsk].
template <typename ET, int D>
__global__ __launch_bounds__(256) void mass_scores_kernel(MassArgs a, float* sc, int stride) {
  using V8 = typename ET::V8;
  constexpr int KS = D / 32, TT = 4, KT = 16 * TT;
  __shared__ float s_m[4][16], s_l[4][16];
  const int hb = (int)blockIdx.x / a.by_nsk, sp = blockIdx.x - hb * a.nsk;
  const int b = hb / a.by_hkv, hk = hb - b * a.Hkv, rows = a.G * a.Tq;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c16 = lane & 15;
  const int r = min(c16, rows - 1), h = r / a.by_tq, t = r - h * a.Tq;
  const int all = (a.Tk + KT - 1) / KT, j0 = part_start(all, sp, a.by_nsk), j1 = part_start(all, sp + 1, a.by_nsk);
  V8 qf[KS];
  const char* qp = a.q + b * a.q_sb + ((long)hk * a.G + h) * a.q_sh + (long)t * a.q_st;
#pragma unroll
  for (int s = 0; s < KS; ++s) qf[s] = load8<V8>(qp + (32 * s + 8 * g) * 2);
  const char* kbase = a.k + b * a.k_sb + hk * a.k_sh;
  V8 kf[TT][KS];
  auto load_keys = [&](int j) {  // (keys behind the sequence are masked, whatever they hold)
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) {
      const char* kp = kbase + (long)min(KT * j + 16 * tt + c16, a.Tk - 1) * a.k_st;
#pragma unroll
      for (int s = 0; s < KS; ++s) kf[tt][s] = load8<V8>(kp + (32 * s + 8 * g) * 2);
    }
  };
  load_keys(j0 + w);  // on their way before the length is known
  const MassSeq sq = mass_seq(a, b);
  const int lim = c16 < rows ? mass_limit(a, sq, t) : 0;
  const int end = min(j1, (sq.len + KT - 1) / KT);  // turns with keys
  float* dst = sc + ((long)hb * rows + c16) * stride;
  float m = kLowest, l = 0.f;
  for (int j = j0 + w; j < end; j += 4) {
    float4_t s[TT];
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) s[tt] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int tt = 0; tt < TT; ++tt) s[tt] = ET::mfma(kf[tt][ks], qf[ks], s[tt]);
    if (j + 4 < end) load_keys(j + 4);
    float mx = m;
#pragma unroll
    for (int i = 0; i < 4 * TT; ++i) {
      const float x = s[i / 4][i % 4] * a.sm_log2;
      s[i / 4][i % 4] = KT * j + 16 * (i / 4) + 4 * g + i % 4 < lim ? x : -INFINITY;
      mx = fmaxf(mx, s[i / 4][i % 4]);
    }
    l *= __builtin_amdgcn_exp2f(m - mx);
    m = mx;
#pragma unroll
    for (int i = 0; i < 4 * TT; ++i) l += __builtin_amdgcn_exp2f(s[i / 4][i % 4] - m);
    if (c16 < rows) {
#pragma unroll
      for (int tt = 0; tt < TT; ++tt) *reinterpret_cast<float4_t*>(dst + KT * j + 16 * tt + 4 * g) = s[tt];
    }
  }
  const float mw = col_max(m), lw = col_sum(l * __builtin_amdgcn_exp2f(m - mw));
  if (g == 0) { s_m[w][c16] = mw; s_l[w][c16] = lw; }
  __syncthreads();
  if ((int)threadIdx.x < rows) {
    float mx = kLowest, ls = 0.f;
    for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s_m[i][threadIdx.x]);
    for (int i = 0; i < 4; ++i) ls += s_l[i][threadIdx.x] * __builtin_amdgcn_exp2f(s_m[i][threadIdx.x] - mx);
    float* p = a.part + 2 * (((long)hb * rows + threadIdx.x) * a.nsk + sp);
    p[0] = mx;
    p[1] = ls;
  }
}

// The weights of those logits: a work-group 1024 keys, a thread four of them.
__global__ __launch_bounds__(256) void mass_weigh_kernel(MassArgs a, const float* sc, int stride) {
  __shared__ float2 s_st[kFewRows];
  const int hb = (int)blockIdx.x / a.by_kpairs, key = (blockIdx.x - hb * a.by_kpairs.d) * 1024 + 4 * (int)threadIdx.x;
  const int b = hb / a.by_hkv, rows = a.G * a.Tq, r = threadIdx.x / 16;
  if (r < rows) {  // (16 lanes a row; a wave's rows that are not there leave it whole groups)
    const float2 st = a.lse ? lse_stat(a.lse[(long)hb * rows + r])
                            : join_parts<16>(reinterpret_cast<const float2*>(a.part) + ((long)hb * rows + r) * a.nsk, a.nsk,
                                             threadIdx.x & 15);
    if (threadIdx.x % 16 == 0) s_st[r] = st;
  }
  __syncthreads();
  const MassSeq sq = mass_seq(a, b);
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (key < sq.len)
    for (int i = 0; i < rows; ++i) {
      const float4_t x = *reinterpret_cast<const float4_t*>(sc + ((long)hb * rows + i) * stride + key);
      const float2 st = s_st[i];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        // (masked: -inf; NaN goes on, but not from a row of infinite lse)
        if (x[u] != -INFINITY && st.y != 0.f) v[u] = fmaf(__builtin_amdgcn_exp2f(x[u] - st.x), st.y, v[u]);
    }
  float* dst = a.out + b * a.o_sb + (hb - b * a.Hkv) * a.o_sh + key;
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (key + u < a.Tk) dst[u] = a.accumulate ? dst[u] + v[u] : v[u];
}

namespace {
int check_mass(const carekv_mass_params* pp) {
  CAREKV_REQUIRE(pp, "null argument");
  const carekv_mass_params& p = *pp;
  CAREKV_REQUIRE(p.head_dim == 64 || p.head_dim == 128, "head_dim must be 64 or 128");
  CAREKV_REQUIRE(p.dtype == CAREKV_F16 || p.dtype == CAREKV_BF16, "dtype must be CAREKV_F16 or CAREKV_BF16");
  CAREKV_REQUIRE(p.batch >= 0 && p.n_queries >= 0 && p.n_keys >= 0, "negative counts");
  CAREKV_REQUIRE(p.n_heads > 0 && p.n_kv_heads > 0 && p.n_heads % p.n_kv_heads == 0,
                 "n_heads must be a positive multiple of n_kv_heads");
  CAREKV_REQUIRE((p.n_queries < 2 || (p.q_st >= 0 && p.q_st < (1 << 22))) &&
                     (p.n_keys < 2 || (p.k_st >= 0 && p.k_st < (1 << 22))),
                 "q and k row strides must be in 0 .. 2^22 elements");
  CAREKV_REQUIRE(p.n_keys < (1 << 30) && (long)p.n_queries * (p.n_heads / p.n_kv_heads) < (1L << 30),
                 "n_keys and the rows of a kv head must be below 2^30");
  return CAREKV_OK;
}

// How a call is cut: the kernel of few rows, or walks.  A causal walk is the
// longer the earlier its key block (the later its row block) lies; the first and
// the last block, the second and the last but one .. make pairs of equal length,
// each cut into equal parts, so that all work-groups end together.
//
// The number of parts that costs least is taken, in times of a tile: a round of
// 512 work-groups (2 a CU) starts in 7 of them; two on a CU take its tiles by
// turns, 2.5 % faster than one alone; the sum of a mass walk's parts costs 3, each
// part that a row's statistics are joined from 0.06.
// Measured (D = 128, 32 / 8 heads, 4 x 64 rows, one WG a CU and tile 1.1 us): K of
// 2048, 1 / 2 / 4 / 8 parts 22.6 / 21.0 / 19.2 / 29.7 us with the sum, of 4096 23.4
// / 24.8 / 32.7, of 8192 32.0 / 42.4; statistics of 1024 keys, 2 / 4 / 8 / 16 parts
// 18.0 / 13.5 / 11.3 / 12.2, of 8192 4 / 8 / 16 / 24 45.7 / 27.9 / 26.5 / 30.4.
struct MassPlan {
  bool few;
  int few_stride;
  int nkb, parts, nqb, nsk;
  bool fold, split;  // split: few rows on many keys, nsk parts
};
int walk_parts(long pairs, long tiles, double sum, double each) {
  long best = 1;
  double least = 1e300;
  for (long p = 1; p <= 64 && (p == 1 || p * 2 <= tiles); ++p) {
    const long wgs = pairs * p;
    const double turns = wgs <= 256 ? 1 : 0.975 * ((wgs + 255) / 256);
    const double c = 7.0 * ((wgs + 511) / 512) + turns * tiles / p + (p > 1 ? sum : 0) + each * p;
    if (c < least) { least = c; best = p; }
  }
  return (int)best;
}
MassPlan mass_plan(const carekv_mass_params& p) {
  MassPlan m{};
  const long G = p.n_heads / p.n_kv_heads, rows = G * p.n_queries, hb = (long)p.batch * p.n_kv_heads;
  m.few_stride = (p.n_keys + 63) / 64 * 64 + 4;
  m.few = rows <= kFewRows && rows * m.few_stride * 4 <= kFewLds && (long)p.n_keys * p.head_dim * 2 <= kFewBytes;
  m.nkb = (p.n_keys + kMassKeys - 1) / kMassKeys;
  m.nqb = (int)((rows + 255) / 256);
  m.parts = m.nsk = 1;
  if (m.few) return m;
  m.split = hb > 0 && rows > 0 && rows <= kFewRows;
  if (m.split) {
    m.few_stride = (p.n_keys + 63) / 64 * 64;
    m.nsk = (int)std::max(1L, std::min({64L, 2048 / hb, ((long)p.n_keys + 255) / 256}));
    return m;
  }
  const long seg = p.n_queries >= 32 ? p.n_queries : rows, nseg = p.n_queries >= 32 ? G : 1;
  const long tiles = (seg + kMassTile - 1) / kMassTile * nseg, ktiles = ((long)p.n_keys + kMassTile - 1) / kMassTile;
  // (a pair of causal walks over as many rows as keys has about the tiles of one whole walk)
  const bool tri = p.causal && 2L * p.n_queries > p.n_keys;
  m.parts = walk_parts(hb * ((m.nkb + 1) / 2), tri || m.nkb == 1 ? tiles : 2 * tiles, 3, 0);
  m.nsk = walk_parts(hb * ((m.nqb + 1) / 2), tri || m.nqb == 1 ? ktiles : 2 * ktiles, 0, 0.06);
  // Few rows' statistics are joined by the mass walks themselves where one round of them is at work and the parts are
  // at most half of a block's K: 4 x 64 rows on 8191 keys, 16 parts, 60.7 us with the 5 us launch, 59.9 without; 1 x 64
  // rows on 8192 keys, 32 parts, 33 with it, 40 without.
  m.fold = rows > 0 && rows <= kFoldRows && rows * m.nsk <= 16 * kFoldRows && hb * ((m.nkb + 1) / 2) * m.parts <= 512;
  return m;
}
long mass_ws(const carekv_mass_params& p, bool have_lse) {
  const MassPlan m = mass_plan(p);
  if (m.few) return 0;
  const long rows = (long)p.batch * p.n_heads * p.n_queries;
  if (m.split) return rows * 4 * (m.few_stride + 2L * m.nsk);
  return (have_lse ? 0 : rows * 8 * (1 + m.nsk)) + (m.parts > 1 ? (long)m.parts * p.batch * p.n_kv_heads * p.n_keys * 4 : 0);
}
}  // namespace

}  // namespace carekv

using namespace carekv;

extern "C" int64_t carekv_attention_mass_workspace_bytes(const carekv_mass_params* pp, int32_t have_lse) {
  if (check_mass(pp) != CAREKV_OK) return -1;
  return mass_ws(*pp, have_lse != 0);
}

extern "C" int carekv_attention_mass(const carekv_mass_params* pp, const void* q, const void* k, const float* lse,
                                     const int32_t* q_start, const int32_t* lengths, float* out, void* workspace,
                                     int64_t workspace_bytes, void* stream) {
  const int rc = check_mass(pp);
  if (rc != CAREKV_OK) return rc;
  const carekv_mass_params& p = *pp;
  if (p.batch == 0 || p.n_keys == 0) return CAREKV_OK;
  CAREKV_REQUIRE(k && out && (workspace || mass_ws(p, lse != nullptr) == 0) && (p.n_queries == 0 || q), "null argument");
  const uintptr_t bits = operand_bits(q, {{p.batch, 2 * p.q_sb}, {p.n_heads, 2 * p.q_sh}, {p.n_queries, 2 * p.q_st}}) |
                         operand_bits(k, {{p.batch, 2 * p.k_sb}, {p.n_kv_heads, 2 * p.k_sh}, {p.n_keys, 2 * p.k_st}}) |
                         (uintptr_t)workspace;
  CAREKV_REQUIRE((bits & 15) == 0, "q and k rows must be 16-byte aligned");
  if (workspace_bytes < mass_ws(p, lse != nullptr)) {
    set_error("carekv_attention_mass: workspace too small (%lld < %lld)", (long long)workspace_bytes,
              (long long)mass_ws(p, lse != nullptr));
    return CAREKV_ESPACE;
  }
  const MassPlan m = mass_plan(p);
  MassArgs a{};
  a.q = (const char*)q; a.k = (const char*)k; a.lse = lse; a.q_start = q_start; a.lengths = lengths; a.q_lengths = p.q_lengths;
  a.out = out;
  a.q_sb = 2 * p.q_sb; a.q_sh = 2 * p.q_sh; a.q_st = p.n_queries > 1 ? 2 * p.q_st : 0; a.k_sb = 2 * p.k_sb; a.k_sh = 2 * p.k_sh;
  a.k_st = p.n_keys > 1 ? 2 * p.k_st : 0; a.o_sb = p.out_sb; a.o_sh = p.out_sh;
  a.B = p.batch; a.Hq = p.n_heads; a.Hkv = p.n_kv_heads; a.G = p.n_heads / p.n_kv_heads; a.Tq = p.n_queries;
  a.Tk = p.n_keys; a.causal = p.causal != 0; a.accumulate = p.accumulate != 0;
  a.nkb = m.nkb; a.parts = m.parts; a.nqb = m.nqb; a.nsk = m.nsk;
  if (p.n_queries >= 32) { a.nseg = a.G; a.seg = a.Tq; }
  else { a.nseg = 1; a.seg = a.G * a.Tq; }
  a.by_nhb = FastDiv((long)p.batch * p.n_kv_heads); a.by_hkv = FastDiv(p.n_kv_heads);
  a.by_tq = FastDiv(std::max(p.n_queries, 1)); a.by_parts = FastDiv(m.parts); a.by_nsk = FastDiv(m.nsk);
  a.by_kpairs = FastDiv((m.nkb + 1) / 2); a.by_qpairs = FastDiv(std::max((m.nqb + 1) / 2, 1));
  a.sm_log2 = (float)((double)p.sm_scale * 1.4426950408889634074);
  const long rows = (long)p.batch * p.n_heads * p.n_queries, hb = (long)p.batch * p.n_kv_heads;
  a.fold = m.fold && !lse;
  a.stat = (float*)workspace;
  a.part = a.stat + (lse ? 0 : 2 * rows);
  a.opart = a.part + (lse ? 0 : 2 * rows * m.nsk);
  if (m.split) {  // the logits, then the parts' statistics
    a.opart = (float*)workspace;
    a.part = a.opart + rows * m.few_stride;
    a.by_kpairs = FastDiv((p.n_keys + 1023) / 1024);
  }
  hipStream_t s = (hipStream_t)stream;
  const long wgs = hb * ((m.nkb + 1) / 2) * m.parts, swgs = hb * ((m.nqb + 1) / 2) * m.nsk, sum = (hb * p.n_keys + 255) / 256;
  CAREKV_REQUIRE(grid_fits(wgs, 512) && grid_fits(swgs, 512) && grid_fits(sum, 256) &&
                     grid_fits((rows + 31) / 32, 256) && grid_fits(m.few ? hb : 0, 1024),
                 "too many blocks");
  return dispatch_elem_d(p.dtype, p.head_dim, [&](auto et, auto d) {
    using ET = decltype(et);
    constexpr int D = decltype(d)::value;
    if (m.few && rows > 0) {
      hipLaunchKernelGGL((mass_few_kernel<ET, D>), dim3((unsigned)hb), dim3(1024), 0, s, a, m.few_stride);
      CAREKV_CHECK_LAUNCH("mass_few");
      return CAREKV_OK;
    }
    if (m.split) {
      hipLaunchKernelGGL((mass_scores_kernel<ET, D>), dim3((unsigned)(hb * m.nsk)), dim3(256), 0, s, a, a.opart, m.few_stride);
      CAREKV_CHECK_LAUNCH("mass_scores");
      hipLaunchKernelGGL(mass_weigh_kernel, dim3((unsigned)(hb * a.by_kpairs.d)), dim3(256), 0, s, a, a.opart, m.few_stride);
      CAREKV_CHECK_LAUNCH("mass_weigh");
      return CAREKV_OK;
    }
    if (!lse && rows > 0) {
      hipLaunchKernelGGL((stats_kernel<ET, D>), dim3((unsigned)swgs), dim3(512), 0, s, a);
      CAREKV_CHECK_LAUNCH("mass_stats");
      if (!a.fold) {
        hipLaunchKernelGGL(mass_join_kernel, dim3((unsigned)((rows + 31) / 32)), dim3(256), 0, s, a);
        CAREKV_CHECK_LAUNCH("mass_join");
      }
    }
    if (lse) hipLaunchKernelGGL((mass_kernel<ET, D, true>), dim3((unsigned)wgs), dim3(512), 0, s, a);
    else hipLaunchKernelGGL((mass_kernel<ET, D, false>), dim3((unsigned)wgs), dim3(512), 0, s, a);
    CAREKV_CHECK_LAUNCH("mass");
    if (a.parts > 1) {
      hipLaunchKernelGGL(mass_sum_kernel, dim3((unsigned)sum), dim3(256), 0, s, a);
      CAREKV_CHECK_LAUNCH("mass_sum");
    }
    return CAREKV_OK;
  });
}
