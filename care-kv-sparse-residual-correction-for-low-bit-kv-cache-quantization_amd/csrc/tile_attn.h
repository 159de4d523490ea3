// The main loop of windowed attention with many rows (window_attention's 16-bit
// rows, paged_attention's 4-bit pages): a work-group has 128 rows of a kv head (4
// waves of 32) and walks over the tiles of 32 keys that any of them sees, K and V
// in LDS (double buffered, one barrier a tile): S^T = K Q^T and O^T += V^T P^T on
// v_mfma_f32_16x16x32, the softmax over a query's column in 32 bits on base-2
// logits.  The weights are rounded to the operands' type (half a step; their sum
// is not), in fp16 against a reference 15 below the row's maximum, so that a weight
// of 2^-29 of the largest is still normal.
//
// Masks are applied where a wave's tile has a key that some row of the wave does
// not see, tiles that none sees are left out.
//
// Bound by products and exponentials, whose times add up more than they overlap: 4
// x 8192 rows of 40 heads, D = 128, window 4096: 2250 - 2410 us, 0.86 - 0.92 PFLOP/s,
// at the 1.7 - 2.0 GHz that the card's power leaves.  Three work-groups a CU, their phases apart, did
// better than 8 waves with 256 rows (3026 us, pages 725 against 570, with values looked at
// as they are stored) and than two tiles on their way with two work-groups a CU (2735);
// 32x32x16 products are slower by themselves (1735 against 1941 TFLOP/s from
// registers).  Short windows add each work-group's start and end: q and the results of
// its 128 rows are as many bytes as 4 tiles of K and V.
#pragma once

#include "rows_attn.h"

namespace carekv {

// Src: where K and V come from.  look says which tile is loaded next, load starts its loads into registers, store
// writes them to LDS (and, where it is to take care, says whether the thread had a V value that is not finite: it writes
// 0 for it, so that a masked weight of 0 times it is no NaN), k_op / v_op read operands, there() tells which halves of the
// tile stored last exist, odd_values() brings the values that are not finite to the rows that see them.
//
// Values are looked at only where a sum came out not finite: the work-group then walks once more, with care.  (Looked at
// as they are stored, they cost every walk: 2530 against 2386 us for 4 x 8192 rows of 40 heads, 138 against 127 for 8
// ragged prompts of 2047.)
template <class Src>
__global__ __launch_bounds__(256, Src::D == 64 ? 4 : 3) void tile_attn_kernel(typename Src::Args a) {
  using ET = typename Src::ET;
  using V8 = typename ET::V8;
  using E = typename Src::Out;
  constexpr int D = Src::D, NQ = 2, QW = 32, QB = 128, KT = 32, KS = D / 32, DT = D / 16;
  constexpr int BUF = Src::kK + Src::kV;
  __shared__ __align__(16) char lds[2 * BUF];
  __shared__ int s_odd[2];  // the last tile in the buffer that held a V value that is not finite
  __shared__ int s_again;
  // the items of a kv head (by_group): a split's blocks side by side, those with more keys first (a block's splits side by
  // side, of which a prompt's short blocks have one or two, load the CUs unevenly: 2 x 1744 rows of 8 heads 38 us, so 33)
  const int it = xcd_item(a), bh = it / a.by_group, in = it - bh * a.by_group.d;
  const int sp = in / a.by_nqb, qblk = a.nqb - 1 - (in - sp * a.nqb);
  const int b = bh / a.by_hkv, hk = bh - b * a.Hkv;
  const int lane = threadIdx.x & 63, g = lane >> 4, c16 = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b0 = qblk * QB, b1 = min(b0 + QB, a.M), r0 = b0 + QW * w, r1 = min(r0 + QW, a.M);
  const SeqRows seq(a, b);
  const Span<KT> span(a, seq, b0 / a.by_g, (b1 - 1) / a.by_g + 1);
  const Span<KT> mine(a, seq, r0 / a.by_g, r1 > r0 ? (r1 - 1) / a.by_g + 1 : 0);
  const int i0 = sp * a.tps, i1 = min(i0 + a.tps, span.n), nt = i1 - i0;
  if (a.nsplit > 1 && nt <= 0) return;  // (the join does not read it)

  if (threadIdx.x < 2) s_odd[threadIdx.x] = -1;
  if (threadIdx.x == 0) s_again = 0;
  V8 qf[NQ][KS];
  float c[NQ];
  RowSight sight[NQ];
#pragma unroll
  for (int qb = 0; qb < NQ; ++qb) {
    sight[qb] = RowSight(a, seq, r0 + 16 * qb + c16);
    c[qb] = Src::load_q(qf[qb], a, b, hk, r0 + 16 * qb + c16, g);
  }
  float m_run[NQ], l_run[NQ];
  float4_t o[NQ][DT];
  Src src(a, b, hk, seq, span.hi, w, lane);
  auto tile = [&](int i) { return span.tile(i0 + i); };
  auto walk = [&](auto with_care) {
    constexpr bool care = decltype(with_care)::value;
#pragma unroll
    for (int qb = 0; qb < NQ; ++qb) {
      m_run[qb] = kLowest;
      l_run[qb] = 0.f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[qb][dt] = float4_t{0.f, 0.f, 0.f, 0.f};
    }
    if (nt > 0) {
      src.look(tile(0));
      src.load();
      src.look(tile(min(1, nt - 1)));
      if (src.template store<care>(lds, lds + Src::kK, tile(0))) s_odd[0] = 0;
    }
    __syncthreads();
    if (nt > 1) src.load();
    for (int i = 0; i < nt; ++i) {
      const int j0 = tile(i) * KT, here = src.there();
      src.look(tile(min(i + 2, nt - 1)));
      const char* kb = lds + (i & 1) * BUF;
      const char* vb = kb + Src::kK;
      if (mine.n > 0 && j0 <= mine.hi && (j0 + KT - 1 > mine.first - a.window || j0 < a.sink)) {
        // (raised wave priority over the products: a wave with products to issue goes before others' softmax)
        __builtin_amdgcn_s_setprio(1);
        float4_t s[2][NQ];
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
#pragma unroll
          for (int qb = 0; qb < NQ; ++qb) s[tt][qb] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            const V8 ak = src.k_op(kb, tt, ks);
#pragma unroll
            for (int qb = 0; qb < NQ; ++qb) s[tt][qb] = ET::mfma(ak, qf[qb][ks], s[tt][qb]);
          }
        }
        __builtin_amdgcn_s_setprio(0);
        if (!mine.whole(a, j0) || here != 3) {
#pragma unroll
          for (int qb = 0; qb < NQ; ++qb) {
            RowSight row = sight[qb];
            row.stay_here();
#pragma unroll
            for (int tt = 0; tt < 2; ++tt)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if (!(here >> tt & 1) || !row.sees(a, j0 + 16 * tt + 4 * g + k)) s[tt][qb][k] = -INFINITY;
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
          over[qb] = fmaf(mx[qb], c[qb], -ET::kUp) > m_run[qb];
          any_over |= over[qb];
        }
        if (__any(any_over)) {
#pragma unroll
          for (int qb = 0; qb < NQ; ++qb) {
            if (!__any(over[qb])) continue;  // columns that keep their reference get a factor of exactly 1
            const float m_new = fmaxf(m_run[qb], fmaf(col_max(mx[qb]), c[qb], -ET::kUp));
            const float f = __builtin_amdgcn_exp2f(m_run[qb] - m_new);
            m_run[qb] = m_new;
            l_run[qb] *= f;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[qb][dt] = care ? rescaled(o[qb][dt], f) : o[qb][dt] * f;
          }
        }
        V8 bp[NQ];
#pragma unroll
        for (int qb = 0; qb < NQ; ++qb) {
          float ls = 0.f;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float p = __builtin_amdgcn_exp2f(fmaf(s[k / 4][qb][k % 4], c[qb], -m_run[qb]));
            ls += p;
            bp[qb][k] = (typename ET::E)p;
          }
          l_run[qb] += ls;
        }
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const V8 av = src.v_op(vb, dt);
#pragma unroll
          for (int qb = 0; qb < NQ; ++qb) o[qb][dt] = ET::mfma(av, bp[qb], o[qb][dt]);
        }
        if (care && s_odd[i & 1] == i) src.odd_values(a, o, sight, tile(i));
      }
      __builtin_amdgcn_s_setprio(0);
      if (i + 1 < nt && src.template store<care>(lds + (i + 1 & 1) * BUF, lds + (i + 1 & 1) * BUF + Src::kK, tile(i + 1)))
        s_odd[(i + 1) & 1] = i + 1;
      if (i + 2 < nt) src.load();
      __syncthreads();
    }
  };
  walk(std::false_type{});
#pragma unroll
  for (int qb = 0; qb < NQ; ++qb) {
    float sum = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int x = 0; x < 4; ++x) sum = fmaf(o[qb][dt][x], 0.f, sum);
    if (!(sum == 0.f) && sight[qb].top >= 0) s_again = 1;
  }
  __syncthreads();
  if (__builtin_expect(s_again, 0)) walk(std::true_type{});

  // the rows' results, or the split's partial (lane: row r0 + 16qb + c16, dims 16dt + 4g ..).  Results go through the
  // wave's part of LDS, 16-byte pieces exchanged against bank conflicts, so that whole rows are written.
  char* turned = lds + w * (QW * 2 * D);
  static_assert(4 * QW * 2 * D <= 2 * BUF, "the waves' results fit the tiles' LDS");
#pragma unroll
  for (int qb = 0; qb < NQ; ++qb) {
    const int r = r0 + 16 * qb + c16;
    const bool pad = sight[qb].top < 0;  // (what a row of padding holds is not used)
    const float l = col_sum(l_run[qb]);
    const float inv = pad || l == 0.f ? 0.f : 1.f / l;
    if (a.nsplit == 1) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        E e[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) e[x] = pad ? (E)0.f : (E)(o[qb][dt][x] * inv);
        __builtin_memcpy(turned + (16 * qb + c16) * (2 * D) + ((2 * dt + (g >> 1)) ^ (c16 & (D / 8 - 1))) * 16 + (g & 1) * 8, e, 8);
      }
    }
    if (r >= a.M) continue;
    if (a.nsplit == 1) {
      if (a.lse && g == 0) write_lse(a, b, hk, r, m_run[qb], pad ? 0.f : l);
    } else {
      const long pr = (long)sp * a.rows + (long)bh * a.M + r;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<float4_t*>(a.po + pr * D + 16 * dt + 4 * g) = o[qb][dt];
      if (g == 0) {
        a.pml[2 * pr] = m_run[qb];
        a.pml[2 * pr + 1] = l;
      }
    }
  }
  if (a.nsplit > 1) return;
  lds_sync_wave();
  constexpr int CH = D / 8, RP = 64 / CH;  // pieces of a row, rows at a time
#pragma unroll
  for (int x = 0; x < QW / RP; ++x) {
    const int row = RP * x + lane / CH, piece = lane % CH, r = r0 + row;
    if (r >= a.M) break;
    typedef uint32_t uint4_v __attribute__((ext_vector_type(4)));
    const uint4_v u = *reinterpret_cast<const uint4_v*>(turned + row * (2 * D) + (piece ^ (row & (CH - 1))) * 16);
    char* dst = out_row(a, b, hk, r) + 16 * piece;
    // (past the L2, where K and V stay: 8 ragged prompts of 2047 tokens replayed in a graph in 140 us, else 152)
    if (a.al16) __builtin_nontemporal_store(u, reinterpret_cast<uint4_v*>(dst));
    else __builtin_memcpy(dst, &u, 16);
  }
}

}  // namespace carekv
