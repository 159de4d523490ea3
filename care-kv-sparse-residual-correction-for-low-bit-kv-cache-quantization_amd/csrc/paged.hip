// Attention of a sequence's last rows over its pages of 4-bit rows
// (paged_attention): o = sum_j e^(s_j) v_j / sum_j e^(s_j), s_j = scale q . k_j,
// over the keys that the row sees (rows_attn.h), k and v the values that the
// pages stand for (pages4.h).
//
// Few rows: bound by reading the pages once.  A work-group has up to 16 NQ rows
// of a kv head and a range of tiles of 32 keys (two pages), its four waves every
// fourth tile; a wave loads a tile's codes and scales straight into the operands'
// lanes, the next tile's while it works on this one, and turns them into fp16
// there.  S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_16x16x32_f16, the softmax over a
// query's column in 32 bits on base-2 logits, the waves joined in LDS.  Measured: 64
// rows of 32 / 8 heads, D = 128, on 32768 keys (2.4 GB) 458 - 470 us, 5.2 TB/s, a copy's
// rate (515 with the table read by vector loads and masks as literals); 16 x 5 rows
// through a window of 4096 33 us, 30 of them this kernel: 20 rows fill 20 of 32 columns,
// and of the 50000 cycles that a wave lives (at some 2 GHz) its SIMD issues vector
// instructions in 33700, 2070 for each of 16.25 tiles (by count unpacking 830, softmax
// and products 510 each), while a wave waits in 18600 of them (all from counters).  One
// row of 32 / 4 heads, D = 64, on 2303 keys in a graph 8.7; with 16 waves a work-group
// and no splits, one launch instead of two, 12.4.
//
// Products are fp16 whatever q's type: codes times scales are fp16 values by
// definition, bf16 rows of q are scaled by a power of two to below 2^12, which
// keeps their 8 bits, and weights are rounded to fp16 (half a step each, 2^-11;
// their sum is not) against a reference 15 below the row's maximum, so that a
// weight of 2^-29 of the largest is still normal.
#include <algorithm>
#include <cmath>

#include "host_util.h"
#include "pages4.h"
#include "tile_attn.h"

namespace carekv {

struct PagedArgs : RowsArgs {
  const int32_t* table;
  const char* pages;
  long table_sb;
  int n_pages, max_pages;
};

constexpr int kTile = 2 * kPage;

// A lane's part of a tile: two pages' codes and scales.
template <int D>
struct Tile4 {
  static constexpr int W = D / 32;  // words of a lane's codes
  uint32_t k[2][W], v[2][W];
  half2_t vs[2][2 * W];             // V scales: group, token pairs
  uint16_t ks[2];
};

// Row r's operand of Q^T (lane group g: dims g D / 4 .., as K's codes lie) in fp16, and its factor on base-2 logits.
template <typename E, int D>
__device__ __forceinline__ float load_q4(half8_t* qf, const RowsArgs& a, int b, int hk, int r, int g) {
  constexpr int KS = D / 32;
  r = min(r, a.M - 1);
  const int t = r / a.by_g, h = hk * a.G + r - t * a.G;
  const char* qp = a.q + b * a.q_sb + h * a.q_sh + t * a.q_st + g * (D / 2);
  uint4 raw[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    uint4 v = *reinterpret_cast<const uint4*>(qp + 16 * s);
    v.x = (v.x ^ a.q_sign) & a.q_keep; v.y = (v.y ^ a.q_sign) & a.q_keep;
    v.z = (v.z ^ a.q_sign) & a.q_keep; v.w = (v.w ^ a.q_sign) & a.q_keep;
    raw[s] = v;
  }
  if constexpr (std::is_same<E, _Float16>::value) {
#pragma unroll
    for (int s = 0; s < KS; ++s) __builtin_memcpy(&qf[s], &raw[s], 16);
    return a.sm_log2;
  } else {
    float x[KS][8], m = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      E e[8];
      __builtin_memcpy(e, &raw[s], 16);
#pragma unroll
      for (int i = 0; i < 8; ++i) { x[s][i] = (float)e[i]; m = fmaxf(m, fabsf(x[s][i])); }
    }
    m = col_max(m);
    int ex = 0;
    if (m > 0.f && m < INFINITY) frexpf(m, &ex), ex -= 12;  // m 2^-ex in [2^11, 2^12)
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int i = 0; i < 8; ++i) qf[s][i] = (_Float16)ldexpf(x[s][i], -ex);
    // (never 0: times the -inf of a key that is not seen it would be no number)
    const float c = ldexpf(a.sm_log2, ex);
    return c < 1.17549435e-38f ? 1.17549435e-38f : c;
  }
}

template <typename E, int D, int NQ>
__global__ __launch_bounds__(256, NQ == 1 ? 3 : 2) void paged_rows_kernel(PagedArgs a) {
  using P = Page4<D>;
  constexpr int W = D / 32, KS = D / 32, DT = D / 16, QB = 16 * NQ;
  constexpr float kUp = ElemF16::kUp;
  const int it = xcd_item(a);
  // a group: the kv heads' blocks of a sequence's split, which lie side by side in its pages
  const int unit = it / a.by_group, b = unit / a.by_nsplit, sp = unit - b * a.nsplit;
  const int in = it - unit * a.by_group.d, hk = in / a.by_nqb, qblk = in - hk * a.nqb, bh = b * a.Hkv + hk;
  const int lane = threadIdx.x & 63, g = lane >> 4, c16 = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r0 = qblk * QB, r1 = min(r0 + QB, a.M);
  const SeqRows seq(a, b);
  const Span<kTile> span(a, seq, r0 / a.by_g, (r1 - 1) / a.by_g + 1);
  const int i0 = sp * a.tps, i1 = min(i0 + a.tps, span.n);
  if (a.nsplit > 1 && i0 >= i1) return;  // (the join does not read it)

  half8_t qf[NQ][KS];
  float c[NQ];
  RowSight sight[NQ];
#pragma unroll
  for (int qb = 0; qb < NQ; ++qb) {
    sight[qb] = RowSight(a, seq, r0 + 16 * qb + c16);
    c[qb] = load_q4<E, D>(qf[qb], a, b, hk, r0 + 16 * qb + c16, g);
  }

  float m_run[NQ], l_run[NQ];
  float4_t o[NQ][DT];
#pragma unroll
  for (int qb = 0; qb < NQ; ++qb) {
    m_run[qb] = kLowest;
    l_run[qb] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[qb][dt] = float4_t{0.f, 0.f, 0.f, 0.f};
  }

  const char* pool = a.pages + (long)hk * P::kBytes;
  const long page_bytes = (long)a.Hkv * P::kBytes;
  // (scalar loads: vector ones come back in order, behind the codes on their way)
  const cint32_t* table = (const cint32_t*)(a.table + b * a.table_sb);
  auto load = [&](Tile4<D>& x, int p0, int p1) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const char* blk = pool + (long)max(i ? p1 : p0, 0) * page_bytes;
      __builtin_memcpy(x.k[i], __builtin_assume_aligned(blk + c16 * (D / 2) + g * 4 * W, 4 * W), 4 * W);
      __builtin_memcpy(x.v[i], __builtin_assume_aligned(blk + P::kV + lane * 4 * W, 4 * W), 4 * W);
      __builtin_memcpy(x.vs[i], __builtin_assume_aligned(blk + P::kVS + g * 8 * W, 16), 8 * W);
      x.ks[i] = *reinterpret_cast<const uint16_t*>(blk + P::kKS + ((D == 128 ? g : g >> 1) * kPage + c16) * 2);
    }
  };

  const Unpack4 dequant4;
  // tile i, whose codes are in cur, of pages p0 and p1
  auto work = [&](Tile4<D>& cur, int p0, int p1, int i) {
    const int j0 = span.tile(i) * kTile;
    float4_t s[2][NQ];
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      const _Float16 ks = bits2half(cur.ks[tt]);
      const half2_t ks2 = {ks, ks}, kss[4] = {ks2, ks2, ks2, ks2};
#pragma unroll
      for (int qb = 0; qb < NQ; ++qb) s[tt][qb] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int st = 0; st < KS; ++st) {
        half2_t kv[4];
        dequant4(kv, cur.k[tt][st], kss);
        half8_t ak;
        __builtin_memcpy(&ak, kv, 16);
#pragma unroll
        for (int qb = 0; qb < NQ; ++qb) s[tt][qb] = mfma16x32(ak, qf[qb][st], s[tt][qb]);
      }
    }
    uint32_t bad[W] = {};  // per group: the lane's keys (page tt, token 4g + k: bit 4 tt + k) that stand for NaN
    const bool whole = span.whole(a, j0) && p0 >= 0 && p1 >= 0;
    uint32_t see[NQ] = {};
    if (!whole) {
      RowSight row[NQ];
#pragma unroll
      for (int qb = 0; qb < NQ; ++qb) {
        row[qb] = sight[qb];
        row[qb].stay_here();
      }
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        const bool there = (tt ? p1 : p0) >= 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int j = j0 + 16 * tt + 4 * g + k;
#pragma unroll
          for (int qb = 0; qb < NQ; ++qb) {
            const bool v = there && row[qb].sees(a, j);
            see[qb] |= (uint32_t)v << (4 * tt + k);
            s[tt][qb][k] = v ? s[tt][qb][k] : -INFINITY;
          }
          // a weight of 0 times a scale that is no number would be NaN: such scales, and what lies where no row looks,
          // are 0 here, and the rows that do see such a key are set below
#pragma unroll
          for (int gr = 0; gr < W; ++gr) {
            _Float16& x = reinterpret_cast<_Float16*>(cur.vs[tt])[4 * gr + k];
            const bool nan = (half2bits(x) & 0x7c00) == 0x7c00;
            if (nan) bad[gr] |= 1u << (4 * tt + k);
            if (nan || !there || j > span.hi) x = (_Float16)0.f;
          }
        }
      }
    }
    float mx[NQ];
    bool any_over = false, over[NQ];
#pragma unroll
    for (int qb = 0; qb < NQ; ++qb) {
      mx[qb] = -INFINITY;
#pragma unroll
      for (int k = 0; k < 8; ++k) mx[qb] = fmaxf(mx[qb], s[k / 4][qb][k % 4]);
      over[qb] = fmaf(mx[qb], c[qb], -kUp) > m_run[qb];
      any_over |= over[qb];
    }
    if (__any(any_over)) {
#pragma unroll
      for (int qb = 0; qb < NQ; ++qb) {
        if (!__any(over[qb])) continue;  // columns that keep their reference get a factor of exactly 1
        const float m_new = fmaxf(m_run[qb], fmaf(col_max(mx[qb]), c[qb], -kUp));
        const float f = __builtin_amdgcn_exp2f(m_run[qb] - m_new);
        m_run[qb] = m_new;
        l_run[qb] *= f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[qb][dt] *= f;
      }
    }
    half8_t bp[NQ];
#pragma unroll
    for (int qb = 0; qb < NQ; ++qb) {
      float ls = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float p = __builtin_amdgcn_exp2f(fmaf(s[k / 4][qb][k % 4], c[qb], -m_run[qb]));
        ls += p;
        bp[qb][k] = (_Float16)p;
      }
      l_run[qb] += ls;
    }
#pragma unroll
    for (int x = 0; x < W; ++x) {  // word x: dims of tiles 2x and 2x + 1, one group
      half2_t v0[4], v1[4];
      const half2_t sc0[4] = {cur.vs[0][2 * x], cur.vs[0][2 * x + 1], cur.vs[0][2 * x], cur.vs[0][2 * x + 1]};
      const half2_t sc1[4] = {cur.vs[1][2 * x], cur.vs[1][2 * x + 1], cur.vs[1][2 * x], cur.vs[1][2 * x + 1]};
      dequant4(v0, cur.v[0][x], sc0);
      dequant4(v1, cur.v[1][x], sc1);
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        half2_t av2[4] = {v0[2 * y], v0[2 * y + 1], v1[2 * y], v1[2 * y + 1]};
        half8_t av;
        __builtin_memcpy(&av, av2, 16);
#pragma unroll
        for (int qb = 0; qb < NQ; ++qb) o[qb][2 * x + y] = mfma16x32(av, bp[qb], o[qb][2 * x + y]);
      }
    }
    if (!whole) {
#pragma unroll
      for (int gr = 0; gr < W; ++gr) {
        if (!__any(bad[gr] != 0)) continue;
#pragma unroll
        for (int qb = 0; qb < NQ; ++qb) {
          const float hit = col_max(bad[gr] & see[qb] ? 1.f : 0.f);
          if (hit > 0.f) o[qb][2 * gr] = o[qb][2 * gr + 1] = float4_t{NAN, NAN, NAN, NAN};
        }
      }
    }
  };
  // the next tile's codes are on their way while one is worked on, two tiles a turn: nothing is moved between them; the
  // pages of the tile behind that are looked up (and checked when they are used: checked at once, they would be waited
  // for at once)
  Tile4<D> x, y;
  int x0 = -1, x1 = -1, y0 = -1, y1 = -1, at, n0, n1;
  auto look = [&](int i) {
    at = 2 * span.tile(max(min(i, i1 - 1), 0));
    n0 = table[min(at, a.max_pages - 1)];
    n1 = table[min(at + 1, a.max_pages - 1)];
  };
  auto checked = [&](int at, int p) { return at < a.max_pages && p >= 0 && p < a.n_pages ? p : -1; };  // -1: not there
  auto fetch = [&](Tile4<D>& t, int& p0, int& p1, int i) {
    if (i >= i1) return;
    p0 = checked(at, n0);
    p1 = checked(at + 1, n1);
    load(t, p0, p1);
    look(i + 4);
  };
  if (i0 < i1) look(i0 + w);
  fetch(x, x0, x1, i0 + w);
  for (int i = i0 + w; i < i1; i += 8) {
    fetch(y, y0, y1, i + 4);
    work(x, x0, x1, i);
    if (i + 4 >= i1) break;
    fetch(x, x0, x1, i + 8);
    work(y, y0, y1, i + 4);
  }

  // the waves' parts of the same rows: (m, l) of every wave, then O scaled to the joint maximum, 16 rows at a time,
  // added in wave order; a wave keeps the dims of tiles w, w + 4 ..
  __shared__ float s_ml[4][QB][2];
  __shared__ __align__(16) float so[4 * DT * 256];  // [waves][DT][64 lanes][4]
#pragma unroll
  for (int qb = 0; qb < NQ; ++qb) {
    const float lt = col_sum(l_run[qb]);
    l_run[qb] = lt;
    if (g == 0) { s_ml[w][16 * qb + c16][0] = m_run[qb]; s_ml[w][16 * qb + c16][1] = lt; }
  }
  __syncthreads();
#pragma unroll
  for (int qb = 0; qb < NQ; ++qb) {
    float m = kLowest, l = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) m = fmaxf(m, s_ml[k][16 * qb + c16][0]);
#pragma unroll
    for (int k = 0; k < 4; ++k) l += s_ml[k][16 * qb + c16][1] * __builtin_amdgcn_exp2f(s_ml[k][16 * qb + c16][0] - m);
    const float f = __builtin_amdgcn_exp2f(m_run[qb] - m);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<float4_t*>(so + ((w * DT + dt) * 64 + lane) * 4) = o[qb][dt] * f;
    __syncthreads();
    const int r = r0 + 16 * qb + c16;
    const bool is_row = r < a.M, pad = sight[qb].top < 0;
#pragma unroll
    for (int u = 0; u < DT / 4; ++u) {
      const int dt = w + 4 * u;
      float4_t v = *reinterpret_cast<const float4_t*>(so + (dt * 64 + lane) * 4);
#pragma unroll
      for (int k = 1; k < 4; ++k) v += *reinterpret_cast<const float4_t*>(so + ((k * DT + dt) * 64 + lane) * 4);
      if (!is_row) continue;
      if (a.nsplit == 1) {
        if (pad) v = float4_t{0.f, 0.f, 0.f, 0.f};
        write4<E>(a, out_row(a, b, hk, r), 16 * dt + 4 * g, v, pad ? 0.f : l);
      } else {
        const long pr = (long)sp * a.rows + (long)bh * a.M + r;
        *reinterpret_cast<float4_t*>(a.po + pr * D + 16 * dt + 4 * g) = v;
      }
    }
    if (is_row && g == 0 && w == 0) {
      if (a.nsplit > 1) {
        const long pr = (long)sp * a.rows + (long)bh * a.M + r;
        a.pml[2 * pr] = m;
        a.pml[2 * pr + 1] = l;
      } else if (a.lse) {
        write_lse(a, b, hk, r, m, pad ? 0.f : l);
      }
    }
    __syncthreads();
  }
}

// Many rows: bound by the products, so that the codes are turned into fp16 once for
// the 128 rows of tile_attn.h.  A wave takes half of one page's codes of a tile of 32
// keys and writes them to LDS as the operands that all four read, 1 KB each in the
// lanes' order.  2 x 512 rows of 40 heads, D = 128, on 16896 keys: 511 - 518 us, 0.68 PFLOP/s.
template <typename E_, int D_>
struct Pages4 {
  using Args = PagedArgs;
  using ET = ElemF16;
  using Out = E_;
  using V8 = half8_t;
  using P = Page4<D_>;
  static constexpr int D = D_, W = D / 32, KS = D / 32, NW = W / 2, kK = 2 * KS * 1024, kV = D / 16 * 1024;
  const char* pool;
  const cint32_t* table;  // (scalar loads)
  long page_bytes;
  int n_pages, max_pages, hi, lane, g, c16, pg, half;  // pg, half: the wave's page of a tile and half of its words
  uint32_t kw[NW], vw[NW];
  half2_t vs[2 * NW];
  uint16_t ks;
  int at, p0, p1;    // the next tile's places in the table and what is there
  int loaded, held;  // which pages of the tile on its way, of the tile stored last, are there: bit i, page i

  __device__ __forceinline__ Pages4(const Args& a, int b, int hk, const SeqRows&, int hi_, int w, int lane_)
      : pool(a.pages + (long)hk * P::kBytes), table((const cint32_t*)(a.table + b * a.table_sb)), page_bytes((long)a.Hkv * P::kBytes),
        n_pages(a.n_pages), max_pages(a.max_pages), hi(hi_), lane(lane_), g(lane_ >> 4), c16(lane_ & 15), pg(w >> 1),
        half(w & 1), loaded(0), held(0) {}
  static __device__ __forceinline__ float load_q(V8* qf, const Args& a, int b, int hk, int r, int g) {
    return load_q4<E_, D>(qf, a, b, hk, r, g);
  }
  __device__ __forceinline__ int checked(int at, int p) const {  // -1: not there
    return at < max_pages && p >= 0 && p < n_pages ? p : -1;
  }
  // (as they are read: checked here, they would be waited for here)
  __device__ __forceinline__ void look(int tile) {
    at = 2 * tile;
    p0 = table[min(at, max_pages - 1)];
    p1 = table[min(at + 1, max_pages - 1)];
  }
  __device__ __forceinline__ void load() {
    const int q0 = checked(at, p0), q1 = checked(at + 1, p1);
    loaded = (q0 >= 0) | (q1 >= 0) << 1;
    const char* blk = pool + (long)max(pg ? q1 : q0, 0) * page_bytes;
    __builtin_memcpy(kw, __builtin_assume_aligned(blk + c16 * (D / 2) + (g * W + half * NW) * 4, 4 * NW), 4 * NW);
    __builtin_memcpy(vw, __builtin_assume_aligned(blk + P::kV + (lane * W + half * NW) * 4, 4 * NW), 4 * NW);
    __builtin_memcpy(vs, __builtin_assume_aligned(blk + P::kVS + (g * W + half * NW) * 8, 8 * NW), 8 * NW);
    ks = *reinterpret_cast<const uint16_t*>(blk + P::kKS + ((D == 128 ? g : g >> 1) * kPage + c16) * 2);
  }
  template <bool CARE>
  __device__ __forceinline__ bool store(char* kb, char* vb, int tile) {
    held = loaded;
    const int j0 = tile * kTile;
    if (j0 + kTile - 1 > hi || held != 3) {  // what lies where no row looks
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (!(held >> pg & 1) || j0 + 16 * pg + 4 * g + k > hi)
#pragma unroll
          for (int x = 0; x < NW; ++x) vs[2 * x + k / 2][k & 1] = (_Float16)0.f;
    }
    bool odd = false;
    if constexpr (CARE) {
#pragma unroll
      for (int x = 0; x < 4 * NW; ++x)
        if ((half2bits(vs[x / 2][x & 1]) & 0x7c00) == 0x7c00) vs[x / 2][x & 1] = (_Float16)0.f, odd = true;
    }
    const Unpack4 dequant4;
    const _Float16 kf = bits2half(ks);
    const half2_t ks2 = {kf, kf}, kss[4] = {ks2, ks2, ks2, ks2};
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      half2_t v[4];
      dequant4(v, kw[x], kss);
      uint4 u;
      __builtin_memcpy(&u, v, 16);
      *reinterpret_cast<uint4*>(kb + (pg * KS + half * NW + x) * 1024 + lane * 16) = u;
      const half2_t sc[4] = {vs[2 * x], vs[2 * x + 1], vs[2 * x], vs[2 * x + 1]};
      dequant4(v, vw[x], sc);
#pragma unroll
      for (int y = 0; y < 2; ++y) {  // four tokens of dims 16 dt + c16: half of an operand
        uint2 t;
        __builtin_memcpy(&t, v + 2 * y, 8);
        *reinterpret_cast<uint2*>(vb + (2 * (half * NW + x) + y) * 1024 + lane * 16 + 8 * pg) = t;
      }
    }
    return odd;
  }
  __device__ __forceinline__ V8 k_op(const char* kb, int tt, int st) const {
    V8 r;
    *reinterpret_cast<uint4*>(&r) = *reinterpret_cast<const uint4*>(kb + (tt * KS + st) * 1024 + lane * 16);
    return r;
  }
  __device__ __forceinline__ V8 v_op(const char* vb, int dt) const {
    V8 r;
    *reinterpret_cast<uint4*>(&r) = *reinterpret_cast<const uint4*>(vb + dt * 1024 + lane * 16);
    return r;
  }
  __device__ __forceinline__ int there() const { return held; }
  // groups that stand for NaN
  template <int NQ, int DT>
  __device__ __forceinline__ void odd_values(const Args& a, float4_t (&o)[NQ][DT], const RowSight (&sight)[NQ], int tile) const {
#pragma unroll 1
    for (int key = 0; key < kTile; ++key) {
      const int i = 2 * tile + key / kPage, p = checked(i, table[min(i, max_pages - 1)]);
      if (p < 0) continue;
      const uint16_t* src = reinterpret_cast<const uint16_t*>(pool + (long)p * page_bytes + P::kVS) + key % 16 / 4 * W * 4 + key % 4;
#pragma unroll
      for (int gr = 0; gr < W; ++gr) {
        asm volatile("" ::: "memory");  // (one at a time: in flight together they would cost the loop its registers)
        if ((src[4 * gr] & 0x7c00) != 0x7c00) continue;
#pragma unroll
        for (int qb = 0; qb < NQ; ++qb) {
          RowSight row = sight[qb];
          row.stay_here();
          if (row.sees(a, kTile * tile + key)) o[qb][2 * gr] += NAN, o[qb][2 * gr + 1] += NAN;
        }
      }
    }
  }
};

namespace {
// How a call is cut: 16 rows of a kv head at once or 32 (up to 64: twice), more in
// blocks of 128, whose splits best_splits gives.  (us, 40 rows of 4 heads as two blocks
// of few and as one of many, D = 64: 64 sequences of 2000 keys 28 / 39, one of 8000 12 /
// 18; of 8 heads, D = 128, on 8000 keys: 64 sequences 288 / 338, 16 89 / 87; 96 rows there
// 129 / 106.)  Key splits of few rows: of at least 8 tiles (two a wave),
// at most 32: the join reads every split's partials.  us a call, by splits: one row of
// 32 / 4 heads, D = 64, on 2303 keys 1 / 4 / 8 / 16 / 32: 17.2 / 10.3 / 9.1 / 8.7 / 9.2, on
// 8000 8 / 16 / 32 / 64: 12.4 / 10.0 / 9.9 / 12.3; 32 / 8 heads, D = 128, on 16000 16 / 32 /
// 64: 16.7 / 14.1 / 16.6; 16 x 5 rows on 8191 through a window of 4096 2 / 4 / 6 / 8: 39 / 34
// / 39 / 39; 64 rows on 32768 1 / 2 / 4 / 6 / 8: 489 / 479 / 461 / 460 / 463.
// Work-groups in all: 512 up to 512 x 64 tiles, then 2048.  us with 512 / 2048, in a graph, below that: 16 x 8 heads, D =
// 128, on 4000 keys 24.5 / 26.8, on 8000 37.8 / 38.6, 5 tokens of each on 7900 46.7 / 59.3, 64 x 4 heads, D = 64, on 3900
// 26.9 / 26.7; above: 64 x 8 heads on 8000 125.9 / 131.1, on 16000 244 / 240, on 32768 489 / 465 (ragged 417 / 342), 64 x 4
// heads, D = 64, on 8000 43.9 / 40.6, on 32000 165 / 144.  For 17 rows and more, two work-groups a CU, the border lies too
// low: 16 x 5 tokens on 8600 49 / 63, on 16000 84 / 101, 64 x 5 on 8000 158 / 176.
// Up to 1024 keys (D = 128: 512) of few rows one split: the join's launch costs the
// host 4 us, its splits save less (one row on 500 keys split 7.9 / 9.3 us on the GPU,
// whole 6.9 / 9.1, with the host 16.8 and 12.6; on 1000 keys 7.9 / 9.3 and 9.9 / 13.1).
struct PagedPlan {
  int nq, nqb, nsplit, tps;  // nq: 16-row sub-blocks, 8 for the kernel of many rows
};
PagedPlan paged_plan(const carekv_paged_params& p) {
  PagedPlan r{};
  const long M = (long)p.seq_len * (p.n_heads / p.n_kv_heads);
  r.nq = M <= 16 ? 1 : M <= 64 ? 2 : 8;
  r.nqb = (int)((M + 16 * r.nq - 1) / (16 * r.nq));
  long keys = (long)p.max_pages * kPage;  // that a block of rows may see
  if (p.window > 0) {
    const long sees = (long)p.window + std::min<long>(p.seq_len, 16L * r.nq) + p.sink + 2 * kTile;
    keys = std::min(keys, sees);
  }
  const long tiles = std::max(1L, (keys + kTile - 1) / kTile), wgs = std::max(1L, (long)p.batch * p.n_kv_heads * r.nqb);
  const double mean = std::min((double)tiles, mean_keys((long)p.max_pages * kPage, p.seq_len, keys) / kTile + 1);
  const long at = wgs * tiles < 512 * 64 ? 512 : 2048;  // work-groups
  const long ns = r.nq == 8 ? best_splits(tiles, mean, wgs, (long)p.batch * p.seq_len * p.n_heads, p.head_dim)
                  : tiles * p.head_dim <= 32 * 64 ? 1 : std::max(1L, std::min(std::min(32L, at / wgs), (tiles + 7) / 8));
  r.tps = (int)((tiles + ns - 1) / ns);
  r.nsplit = (int)((tiles + r.tps - 1) / r.tps);
  return r;
}
long paged_ws(const carekv_paged_params& p, const PagedPlan& r) {
  const long rows = (long)p.batch * p.seq_len * p.n_heads;
  return r.nsplit > 1 ? r.nsplit * rows * (2 + p.head_dim) * 4 : 0;
}
int check_paged(const carekv_paged_params* pp) {
  CAREKV_REQUIRE(pp, "null argument");
  const carekv_paged_params& p = *pp;
  CAREKV_REQUIRE(p.head_dim == 64 || p.head_dim == 128, "head_dim must be 64 or 128");
  CAREKV_REQUIRE(p.dtype == CAREKV_F16 || p.dtype == CAREKV_BF16, "dtype must be CAREKV_F16 or CAREKV_BF16");
  CAREKV_REQUIRE(p.batch >= 0 && p.seq_len >= 0 && p.n_pages >= 0 && p.max_pages >= 0 && p.window >= 0 && p.sink >= 0,
                 "negative counts");
  CAREKV_REQUIRE(p.n_heads > 0 && p.n_kv_heads > 0 && p.n_heads % p.n_kv_heads == 0,
                 "n_heads must be a positive multiple of n_kv_heads");
  CAREKV_REQUIRE((long)p.batch * p.seq_len * p.n_heads < (1L << 30), "too many rows");
  CAREKV_REQUIRE(p.max_pages < kMaxPos / kPage && p.seq_len < kMaxPos, "max_pages must be below 2^25, seq_len below 2^29");
  return CAREKV_OK;
}
}  // namespace

}  // namespace carekv

using namespace carekv;

extern "C" int64_t carekv_paged_attn_workspace_bytes(const carekv_paged_params* pp) {
  if (check_paged(pp) != CAREKV_OK) return -1;
  return paged_ws(*pp, paged_plan(*pp));
}

extern "C" int carekv_paged_attn(const carekv_paged_params* pp, const void* q, const void* pages, const int32_t* table,
                                 const int32_t* lengths, const int32_t* q_lengths, void* out, float* lse,
                                 void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = check_paged(pp);
  if (rc != CAREKV_OK) return rc;
  const carekv_paged_params& p = *pp;
  const long rows = (long)p.batch * p.seq_len * p.n_heads;
  if (rows == 0) return CAREKV_OK;
  const PagedPlan plan = paged_plan(p);
  CAREKV_REQUIRE(q && out && lengths && (p.max_pages == 0 || table) && (p.n_pages == 0 || pages) &&
                     (workspace || plan.nsplit < 2), "null argument");
  const uintptr_t bits = operand_bits(q, {{p.batch, 2 * p.q_sb}, {p.n_heads, 2 * p.q_sh}, {p.seq_len, 2 * p.q_st}}) |
                         (uintptr_t)pages | (uintptr_t)workspace;
  CAREKV_REQUIRE((bits & 15) == 0, "rows of q, pages and workspace must be 16-byte aligned");
  if (workspace_bytes < paged_ws(p, plan)) {
    set_error("carekv_paged_attn: workspace too small (%lld < %lld)", (long long)workspace_bytes, (long long)paged_ws(p, plan));
    return CAREKV_ESPACE;
  }
  PagedArgs a{};
  a.q = (const char*)q; a.out = (char*)out; a.lse = lse; a.lengths = lengths; a.q_lengths = q_lengths;
  a.q_sb = 2 * p.q_sb; a.q_sh = 2 * p.q_sh; a.q_st = 2 * p.q_st; a.o_sb = 2 * p.out_sb; a.o_sh = 2 * p.out_sh; a.o_st = 2 * p.out_st;
  a.Hq = p.n_heads; a.Hkv = p.n_kv_heads; a.G = p.n_heads / p.n_kv_heads; a.T = p.seq_len; a.M = a.G * p.seq_len;
  a.rows = rows;
  // without pages nothing is there to be seen
  a.max_keys = p.n_pages == 0 ? 0 : p.max_pages * kPage;
  a.window = p.window > 0 ? std::min(p.window, 2 * kMaxPos) : 2 * kMaxPos;
  a.sink = p.sink;
  a.nqb = plan.nqb; a.nsplit = plan.nsplit; a.tps = plan.tps; a.qb_rows = 16 * plan.nq;
  a.by_g = FastDiv(a.G); a.by_nqb = FastDiv(a.nqb); a.by_hkv = FastDiv(a.Hkv); a.by_nsplit = FastDiv(a.nsplit); a.by_m = FastDiv(a.M);
  if (plan.nq == 8) set_groups(a, (long)a.nqb * a.nsplit, (long)p.batch * a.Hkv);
  else set_groups(a, (long)a.nqb * a.Hkv, (long)p.batch * a.nsplit);
  a.po = (float*)workspace;
  a.pml = a.po + plan.nsplit * rows * p.head_dim;
  set_scale(a, p.sm_scale);
  set_period(a, p.window, (a.qb_rows + a.G - 1) / a.G, kTile);
  set_alignment(a, p.batch);
  a.table = table; a.pages = (const char*)pages; a.table_sb = p.table_sb; a.n_pages = p.n_pages; a.max_pages = p.max_pages;
  hipStream_t s = (hipStream_t)stream;
  const long wgs = (long)p.batch * a.Hkv * a.nqb * a.nsplit;
  CAREKV_REQUIRE(grid_fits(wgs, 256) && grid_fits(rows / (256 / p.head_dim) + 1, 256), "too many rows");
  return dispatch_elem_d(p.dtype, p.head_dim, [&](auto et, auto d) {
    using E = typename decltype(et)::E;
    constexpr int D = decltype(d)::value;
    const dim3 grid((unsigned)wgs), block(256);
    if (plan.nq == 1) hipLaunchKernelGGL((paged_rows_kernel<E, D, 1>), grid, block, 0, s, a);
    else if (plan.nq == 2) hipLaunchKernelGGL((paged_rows_kernel<E, D, 2>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((tile_attn_kernel<Pages4<E, D>>), grid, block, 0, s, a);
    CAREKV_CHECK_LAUNCH("paged_rows");
    if (a.nsplit > 1) {
      launch_join<E, D, kTile>(a, s);
      CAREKV_CHECK_LAUNCH("rows_join");
    }
    return CAREKV_OK;
  });
}
