// What the rows of windowed attention see (paged_attention, window_attention),
// and how parts of their keys are joined.
//
// Query row t of sequence b, t < q_lengths[b], stands at position p = q_start[b]
// + t and sees the keys j <= p, j < lengths[b], with j > p - window or j < sink.
// The rows of a kv head are numbered r = t G + h over its G query heads, so that
// rows next to each other see nearly the same keys.
#pragma once

#include <algorithm>
#include <cmath>

#include "fast_div.h"
#include "mfma16.h"

namespace carekv {

constexpr int kMaxPos = 1 << 29;  // keys, query rows and the distance of q_start from 0 are below it, a window at most twice

struct RowsArgs {
  const char* q;
  char* out;
  float* lse;                // [B][Hq][T], or null
  const int32_t* lengths;    // or null: max_keys
  const int32_t* q_lengths;  // or null: T
  const int32_t* q_start;    // or null: the rows are the sequence's last
  float* pml;                // [nsplit][rows][2] reference (base 2), sum
  float* po;                 // [nsplit][rows][D]
  long q_sb, q_sh, q_st, o_sb, o_sh, o_st;  // bytes
  long rows;                 // B * Hkv * M
  int Hq, Hkv, G, T, M, max_keys, window, sink, nqb, nsplit, qb_rows;
  int tps;                   // tiles of a split
  FastDiv by_g, by_nqb, by_hkv, by_nsplit, by_m;
  FastDiv by_group, by_left; // items of a group, groups that eight does not divide (see xcd_item)
  FastDiv by_period;         // tiles of a window and a block's tokens (see Span)
  float sm_log2;             // |scale| log2(e), 1 where that is 0
  uint32_t q_sign, q_keep;   // sign bits of two elements where the scale is negative; 0 where it is 0
  int al8, al16;             // rows of out on 8, on 16 bytes
};

// The work-group's item.  Items come in groups of a.by_group that read the same
// memory; work-groups go round the 8 XCDs, and an XCD takes one group of every
// eight, each time another one of them, so that the items of a group meet in its
// L2 and each XCD has some of every (ragged) sequence (8 ragged prompts of 2047 tokens
// 159 us, in plain order 208).  The up to seven groups that are left over go side by
// side, longest items first, over all XCDs (8192 rows of 4 kv heads, D = 64: 339 us, one
// after the other 405, a part of them to each XCD 449).
// Blocks of 2 to 8 heads in turn, longest first: full 8192 rows 2 % better, through a
// window the same, ragged batches up to a fifth worse.
__device__ __forceinline__ int xcd_item(const RowsArgs& a) {
  const int idx = blockIdx.x, n = gridDim.x, x = idx & 7, per = a.by_group.d;
  const int whole = n / a.by_group / 8 * 8 * per;
  if (idx < whole) {
    const int j = (idx >> 3) / a.by_group;
    return (8 * j + (x + j & 7)) * per + (idx >> 3) - j * per;
  }
  const int j = idx - whole, at = j / a.by_left;
  return whole + (j - at * a.by_left.d) * per + at;
}

// Sequence b's counts, kept where sums of them stay in 32 bits.
struct SeqRows {
  int len, qlen, base;  // keys, rows that are no padding, position of row 0
  __device__ __forceinline__ SeqRows(const RowsArgs& a, int b) {
    len = a.lengths ? min(max(a.lengths[b], 0), a.max_keys) : a.max_keys;
    qlen = a.q_lengths ? min(max(a.q_lengths[b], 0), a.T) : a.T;
    base = a.q_start ? min(max(a.q_start[b], -kMaxPos), kMaxPos) : len - qlen;
  }
};

// The keys that rows t0 .. t1 - 1 see between them, as tiles of KT keys: the
// first n_sink tiles, then those from tile0 on, begun at the multiple of the
// period among them: blocks that run side by side then read the same one or two
// tiles at a time whatever their windows start with, and those come from the L2.
template <int KT>
struct Span {
  int first, last;  // positions of the first and the last row
  int hi;           // last key that is seen
  int n_sink, tile0, n_main, turn, n;
  __device__ __forceinline__ Span(const RowsArgs& a, const SeqRows& s, int t0, int t1) {
    t1 = min(t1, s.qlen);
    first = s.base + t0;
    last = s.base + t1 - 1;
    hi = min(last, s.len - 1);
    n_sink = tile0 = n_main = turn = n = 0;
    if (t0 >= t1 || hi < 0) return;
    tile0 = max(0, first - a.window + 1) / KT;
    n_sink = min((min(a.sink, hi + 1) + KT - 1) / KT, tile0);
    n_main = max(0, hi / KT - tile0 + 1);
    n = n_sink + n_main;
    turn = (tile0 + a.by_period.d - 1) / a.by_period * a.by_period.d - tile0;
    if (turn >= n_main) turn = 0;
  }
  __device__ __forceinline__ int tile(int i) const {
    const int j = i - n_sink + turn;
    return i < n_sink ? i : tile0 + (j < n_main ? j : j - n_main);
  }
  // whether every row sees every key of the tile at j0
  __device__ __forceinline__ bool whole(const RowsArgs& a, int j0) const {
    return j0 + KT - 1 <= min(first, hi) && (j0 > last - a.window || j0 + KT <= a.sink);
  }
};

// Position of row r, below every key where it is padding or there is none; and its bounds: the row sees key j where
// j <= top and (j >= low or j < sink).
struct RowSight {
  int top, low;
  RowSight() = default;
  __device__ __forceinline__ RowSight(const RowsArgs& a, const SeqRows& s, int r) {
    const int t = r / a.by_g;
    const bool there = r < a.M && t < s.qlen;
    top = there ? min(s.base + t, s.len - 1) : -1;
    low = s.base + t - a.window + 1;
  }
  // in a branch that few tiles take: without it the compiler compares for every tile
  __device__ __forceinline__ void stay_here() { asm volatile("" : "+v"(top), "+v"(low)); }
  __device__ __forceinline__ bool sees(const RowsArgs& a, int j) const { return j <= top && (j >= low || j < a.sink); }
};

// Row r of kv head hk of sequence b: where its output starts, and its place in lse.
__device__ __forceinline__ char* out_row(const RowsArgs& a, int b, int hk, int r) {
  const int t = r / a.by_g, h = hk * a.G + r - t * a.G;
  return a.out + b * a.o_sb + h * a.o_sh + t * a.o_st;
}
__device__ __forceinline__ void write_lse(const RowsArgs& a, int b, int hk, int r, float m, float l) {
  const int t = r / a.by_g, h = hk * a.G + r - t * a.G;
  a.lse[((long)b * a.Hq + h) * a.T + t] = l == 0.f ? -INFINITY : (m + __log2f(l)) * kLn2;
}
// A row's sums under a new reference.  What is not finite stays as it is: an infinity that a row sees is its result however
// small its weight, and 0 times it, where f is that small, would be no number.
__device__ __forceinline__ float4_t rescaled(float4_t o, float f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = fabsf(o[i]) < INFINITY ? o[i] * f : o[i];
  return o;
}
__device__ __forceinline__ bool all_finite(float4_t o) {
  return fmaf(o[0], 0.f, fmaf(o[1], 0.f, fmaf(o[2], 0.f, o[3] * 0.f))) == 0.f;
}
// four neighbouring dims of a row, o / l (0 for a row that sees nothing)
template <typename E>
__device__ __forceinline__ void write4(const RowsArgs& a, char* row, int d, float4_t o, float l) {
  const float inv = l == 0.f ? 0.f : 1.f / l;
  E w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = (E)(o[i] * inv);
  E* dst = reinterpret_cast<E*>(row) + d;
  if (a.al8) __builtin_memcpy(__builtin_assume_aligned(dst, 8), w, 8);
  else
#pragma unroll
    for (int i = 0; i < 4; ++i) dst[i] = w[i];
}

// The splits' partials of a row: D / 4 threads a row for up to 8 splits, else JG = 4
// groups of them that take every fourth split, added up in LDS in group order.  Splits
// behind the rows' last tile wrote nothing and are not read.  Sums that come out not
// finite are added up once more, by what rescaled does (in every sum it cost one row on
// 2303 keys 0.7 us, so 0.1).  4 - 5 us for the rows of single tokens; 40960 rows of 4
// splits (95 MB) 18, with the groups 27.
template <typename E, int D, int KT, int JG>
__global__ __launch_bounds__(256) void rows_join_kernel(RowsArgs a) {
  constexpr int D4 = D / 4, RW = 256 / (D4 * JG);
  const int d4 = threadIdx.x % D4, grp = threadIdx.x / D4 % JG, rw = threadIdx.x / (D4 * JG);
  const long pr = (long)blockIdx.x * RW + rw;
  const bool in = pr < a.rows;
  float m = kLowest, L = 0.f;
  float4_t o = {0.f, 0.f, 0.f, 0.f};
  int b = 0, hk = 0, r = 0;
  bool pad = false;
  if (in) {
    const int bh = (int)pr / a.by_m;
    r = (int)pr - bh * a.M;
    b = bh / a.by_hkv;
    hk = bh - b * a.Hkv;
    const SeqRows s(a, b);
    const int r0 = r / a.qb_rows * a.qb_rows, r1 = min(r0 + a.qb_rows, a.M);
    const Span<KT> span(a, s, r0 / a.by_g, (r1 - 1) / a.by_g + 1);
    const int ns = (span.n + a.tps - 1) / a.tps;
    pad = r / a.by_g >= s.qlen;
    auto add_up = [&](auto with_care) {
      m = kLowest;
      L = 0.f;
      o = float4_t{0.f, 0.f, 0.f, 0.f};
      for (int s0 = grp; s0 < ns; s0 += 4 * JG) {  // four splits' loads in flight
        float2 ml[4];
        float4_t v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const long at = min(s0 + u * JG, ns - 1) * a.rows + pr;
          ml[u] = *reinterpret_cast<const float2*>(a.pml + 2 * at);
          v[u] = *reinterpret_cast<const float4_t*>(a.po + at * D + 4 * d4);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (s0 + u * JG >= ns) break;
          const float mn = fmaxf(m, ml[u].x), f = __builtin_amdgcn_exp2f(m - mn), e = __builtin_amdgcn_exp2f(ml[u].x - mn);
          o = decltype(with_care)::value ? rescaled(o, f) + rescaled(v[u], e) : o * f + v[u] * e;
          L = L * f + ml[u].y * e;
          m = mn;
        }
      }
    };
    add_up(std::false_type{});
    if (__builtin_expect(!all_finite(o), 0)) add_up(std::true_type{});
  }
  if constexpr (JG > 1) {
    __shared__ float4_t s_o[256];
    __shared__ float2 s_ml[RW][JG];
    s_o[threadIdx.x] = o;
    if (d4 == 0) s_ml[rw][grp] = make_float2(m, L);
    __syncthreads();
    m = kLowest;
    L = 0.f;
    o = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < JG; ++i) m = fmaxf(m, s_ml[rw][i].x);
#pragma unroll
    for (int i = 0; i < JG; ++i) {
      const float f = __builtin_amdgcn_exp2f(s_ml[rw][i].x - m);
      L += s_ml[rw][i].y * f;
      o += s_o[(rw * JG + i) * D4 + d4] * f;
    }
    if (__builtin_expect(!all_finite(o), 0)) {
      o = float4_t{0.f, 0.f, 0.f, 0.f};
      for (int i = 0; i < JG; ++i) o += rescaled(s_o[(rw * JG + i) * D4 + d4], __builtin_amdgcn_exp2f(s_ml[rw][i].x - m));
    }
  }
  if (!in || grp != 0) return;
  if (pad) { L = 0.f; o = float4_t{0.f, 0.f, 0.f, 0.f}; }  // (what a row of padding holds is not used)
  write4<E>(a, out_row(a, b, hk, r), 4 * d4, o, L);
  if (a.lse && d4 == 0) write_lse(a, b, hk, r, m, L);
}

template <typename E, int D, int KT>
inline void launch_join(const RowsArgs& a, hipStream_t s) {
  auto go = [&](auto jg) {
    constexpr int JG = decltype(jg)::value, RW = 1024 / (D * JG);
    hipLaunchKernelGGL((rows_join_kernel<E, D, KT, JG>), dim3((unsigned)((a.rows + RW - 1) / RW)), dim3(256), 0, s, a);
  };
  if (a.nsplit <= 8) go(std::integral_constant<int, 1>{});
  else go(std::integral_constant<int, 4>{});
}

// Keys that a row sees on average: the last `rows` positions of `keys`, each those up to itself, at most `most`.
inline double mean_keys(long keys, long rows, long most) {
  const double m = (double)most;
  auto area = [&](double x) { return x <= m ? x * x / 2 : m * m / 2 + m * (x - m); };
  return (area((double)keys) - area((double)std::max(0L, keys - rows))) / (double)std::max(1L, rows);
}

// Key splits of a call of many rows (at most `tiles` tiles of 32 keys for each of `wgs` work-groups, `mean` on average): of
// 1 to 32 the number with the smallest estimate of its time.  Work-groups, longest first, fill the places (4 a CU at D = 64,
// 3 at 128): the longest of them, or their sum over the places, and where they are alike what the last round leaves empty.
// Two and more splits cost the join and the partials, and have to be a tenth better than one.  Over 29 shapes it takes 0.9 %
// more on average than the best number, at most 9.5 % (with whole rounds of work-groups that all have `tiles` 3.4 and 23: a
// prompt's have half of them).  us by splits: 2 x 512 rows of 40 heads on 16896 keys 1 / 2 / 4 / 7 / 8: 837 / 530 / 516 /
// 516 / 532; 4 x 64 rows of 32 / 8 heads on 8000 5 / 8 / 12 / 16: 104 / 76 / 73 / 93; prompts, 1 / 2 / 3: 512 tokens of 40
// heads 26 / 31 / 30, 4096 of 32 / 8 173 / 210 / 212 (3: 195 MB of partials), 8192 of 40 812 / 850 / 884 (2: 325 MB).
inline long best_splits(long tiles, double mean, long wgs, long rows, int d) {
  const double places = d == 64 ? 1024 : 768;
  const double tile = d == 64 ? 0.8 : 1.3, start = 6.0, join = 12.0, split = rows * (d + 2) * 4 / 3.5e6;  // us
  long best = 1;
  double least = 0.0;
  for (long ns = 1; ns <= std::min(tiles, 32L); ++ns) {
    const long tps = (tiles + ns - 1) / ns;
    const double used = std::min((double)ns, std::max(1.0, mean / tps + 0.5)), items = wgs * used;  // splits that have tiles
    const double longest = tps * tile + start, sum = wgs * mean * tile + items * start;
    const double alike = std::max(0.0, 2 * sum / (items * longest) - 1);  // 0 for a prompt's, 1 where all are as long
    const double fill = sum / places + alike * longest * (std::ceil(items / places) - items / places);
    const double cost = std::max(longest, fill) + (ns > 1 ? join + used * split : 0.0);
    if (ns == 1) least = 0.9 * cost;
    else if (cost < least) least = cost, best = ns;
  }
  return best;
}

// Whether rows of out lie on 8 and on 16 bytes.
inline void set_alignment(RowsArgs& a, int batch) {
  const uintptr_t bits = operand_bits(a.out, {{batch, a.o_sb}, {a.Hq, a.o_sh}, {a.T, a.o_st}});
  a.al8 = (bits & 7) == 0;
  a.al16 = (bits & 15) == 0;
}

// The groups of a launch, of `per` items each.
inline void set_groups(RowsArgs& a, long per, long groups) {
  a.by_group = FastDiv(per);
  a.by_left = FastDiv(std::max(1L, groups % 8));
}

// The period of blocks of `tokens` tokens and tiles of kt keys.
inline void set_period(RowsArgs& a, int window, int tokens, int kt) {
  a.by_period = FastDiv(window > 0 ? std::min(((long)window + tokens) / kt + 2, (long)kMaxPos) : kMaxPos);
}

// The scale as the kernels take it.
inline void set_scale(RowsArgs& a, float scale) {
  a.sm_log2 = (float)(std::fabs((double)scale) * 1.4426950408889634074);
  a.q_sign = scale < 0.f ? 0x80008000u : 0u;
  a.q_keep = a.sm_log2 == 0.f ? 0u : ~0u;
  if (a.sm_log2 == 0.f) a.sm_log2 = 1.f;
}

}  // namespace carekv
