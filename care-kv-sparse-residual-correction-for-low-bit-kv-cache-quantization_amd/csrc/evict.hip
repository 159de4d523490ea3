// Rows of a K/V prompt kept by weight (evict_rows): per (sequence, kv head)
// the first `sink` and last `recent` rows, then the rows of largest weight
// (equal weights: the lower index), `keep` in all, in index order; their K, V
// and weight rows gathered.
//
// Weights are mapped to unsigned keys of the same order (NaN to 0, below -inf);
// three histograms of 11, 11 and 10 bits find the key of the last kept row and
// how many of its equals are kept; a scan in index order places the kept rows.
//
// Up to 16384 rows: evict_select_kernel, one work-group a (sequence, kv head),
// the keys in registers (8 a thread, past 8192 rows 16), everything in one launch,
// small results gathered there too.  Longer: the rows are cut into parts of 8192 (at most 64 parts), a
// work-group each, and every histogram is a launch (evict_part_kernel): each
// part writes its own, the next launch adds up its row's, so that nothing is
// cleared and no sum depends on an order.  evict_gather_kernel copies the rows.
//
// Bound by memory: each weight and kept row read once, each kept row written;
// the select is a chain of latencies.  Measured: 16 rows of 131072 weights, 16384
// kept (279 MB): select 35 us in four launches (one work-group a row 251), gather
// 45 us, 6.0 TB/s; 64 rows of 8192, 2048 kept (137 MB): 12.8 + 22 us; 4 rows of
// 512 10 us in one launch.  One launch or four and the gather, in a graph: 4 rows of
// 12000, 1024 kept 17.7 / 27.8 us, 64 of 16384, 4096 kept 59 / 67, 512 of 9000, 1024
// kept 145 / 198; with 32 keys a thread 4 rows of 24000 30.3, in four 28.8.
#include <algorithm>

#include "common.h"
#include "fast_div.h"
#include "host_util.h"

namespace carekv {

struct EvictArgs {
  const char* mass;
  const char* k;
  const char* v;
  const int32_t* lengths;
  char* ko;
  char* vo;
  float* mo;
  int32_t* index;
  int32_t* kept;
  long m_sb, m_sh, k_sb, k_sh, k_st, v_sb, v_sh, v_st;  // bytes
  int H, T, keep, sink, recent, row_bytes;
  FastDiv by_h, by_parts, by_per;  // per: threads of a kept row
};

// unsigned order of a weight: -inf < finite < +inf as unsigned integers, NaN lowest
__device__ __forceinline__ uint32_t weight_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);  // (-0 counts as +0)
  if (x != x) return 0u;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSel = 1024;           // threads of a select work-group
constexpr int kEpt = 8;              // keys a thread holds, or twice as many of rows in one launch
constexpr int kChunk = kSel * kEpt;  // rows of a part's turn
constexpr int kBins = 2048;
constexpr int kMaxParts = 64;
constexpr long kFuseBytes = 65536;   // K rows of a kv head gathered by the select work-group itself

__device__ __forceinline__ int pass_shift(int pass) { return pass == 0 ? 21 : pass == 1 ? 10 : 0; }
__device__ __forceinline__ int pass_bins(int pass) { return pass == 2 ? 1024 : 2048; }

// The rows of a sequence: kept for certain below lo and from hi on, `need` of
// those between by weight; none competes where every row is kept.
struct EvictSeq {
  int n, kept, lo, hi, need;
};
__device__ __forceinline__ EvictSeq evict_seq(const EvictArgs& a, int b) {
  EvictSeq s;
  s.n = a.lengths ? min(max(a.lengths[b], 0), a.T) : a.T;
  s.kept = min(s.n, a.keep);
  if (s.n <= a.keep) {
    s.lo = s.n; s.hi = s.n; s.need = 0;
  } else {
    s.lo = min(a.sink, s.n);
    s.hi = max(s.n - a.recent, s.lo);
    s.need = s.kept - s.lo - (s.n - s.hi);
  }
  return s;
}

struct SelectScratch {
  int part[kSel / 64], part2[kSel / 64], bin, need;
};

// Exclusive prefix over the work-group of (x, y) in thread order, and the totals.
__device__ __forceinline__ void block_scan2(int& x, int& y, int& tx, int& ty, SelectScratch& sc) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, x0 = x, y0 = y;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(x, o, 64), v = __shfl_up(y, o, 64);
    if (lane >= o) { x += u; y += v; }
  }
  if (lane == 63) { sc.part[w] = x; sc.part2[w] = y; }
  __syncthreads();
  int bx = 0, by = 0;
  tx = ty = 0;
#pragma unroll
  for (int i = 0; i < kSel / 64; ++i) {
    if (i < w) { bx += sc.part[i]; by += sc.part2[i]; }
    tx += sc.part[i];
    ty += sc.part2[i];
  }
  x += bx - x0;
  y += by - y0;
  __syncthreads();
}

// The bin, from the top, where the counts pass `need`, and what is left of
// need in it.  Thread t holds the counts c0, c1 of bins nb-1-2t, nb-2-2t (0
// past the bins).
__device__ __forceinline__ void find_bin(int c0, int c1, int nb, int need, int& bin, int& left, SelectScratch& sc) {
  int before = c0 + c1, zero = 0, t0, t1;
  block_scan2(before, zero, t0, t1, sc);
  if (before < need && need <= before + c0 + c1) {
    const bool second = need > before + c0;
    sc.bin = nb - 1 - 2 * (int)threadIdx.x - (second ? 1 : 0);
    sc.need = need - before - (second ? c0 : 0);
  }
  __syncthreads();
  bin = sc.bin;
  left = sc.need;
}

// find_bin by one wave over counts in LDS: each lane adds up a run of bins from
// the top, then the lanes share the bins of the run that passes `need`.
__device__ __forceinline__ void find_bin_wave(const int* hist, int nb, int need, SelectScratch& sc) {
  const int lane = threadIdx.x & 63, per = nb / 64;  // 32 or 16 bins
  auto scan = [&](int c) {
    int x = c;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(x, o, 64);
      if (lane >= o) x += y;
    }
    return x - c;
  };
  int c = 0;
  for (int i = 0; i < per; i += 4) {
    const int4 v = *reinterpret_cast<const int4*>(hist + nb - (lane + 1) * per + i);
    c += v.x + v.y + v.z + v.w;
  }
  const int before = scan(c);
  const int run = __ffsll((unsigned long long)__ballot(before < need && need <= before + c)) - 1;
  const int left = need - __shfl(before, run, 64);
  const int bin = nb - 1 - run * per - lane, d = lane < per ? hist[bin] : 0, b2 = scan(d);
  if (b2 < left && left <= b2 + d) {
    sc.bin = bin;
    sc.need = left - b2;
  }
}

// Row e of this thread in a turn that starts at c0: a wave's loads are consecutive rows.
template <int EPT>
__device__ __forceinline__ int turn_row(int c0, int e) {
  return c0 + (int)(threadIdx.x >> 6) * 64 * EPT + 64 * e + (int)(threadIdx.x & 63);
}

// Places of a turn's rows, given their keys, in index order: those kept for
// certain or above thr, and the first `left` of its equals.  base: places taken
// before the turn, eqb: equals seen before it.
template <int EPT, typename F>
__device__ __forceinline__ void place_rows(const EvictSeq& q, const uint32_t (&key)[EPT], int c0, int end, uint32_t thr,
                                           int left, int& base, int& eqb, SelectScratch& sc, F&& put) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  uint64_t sure[EPT], eq[EPT];
  int ts = 0, te = 0;
#pragma unroll
  for (int e = 0; e < EPT; ++e) {
    const int i = turn_row<EPT>(c0, e);
    const bool in = i < end, by = in && i >= q.lo && i < q.hi;
    sure[e] = __ballot((in && !by) || (by && q.need > 0 && key[e] > thr));
    eq[e] = __ballot(by && q.need > 0 && key[e] == thr);
    ts += __popcll(sure[e]);
    te += __popcll(eq[e]);
  }
  if (lane == 0) { sc.part[w] = ts; sc.part2[w] = te; }
  __syncthreads();
  int s0 = base, e0 = eqb, all_s = 0, all_e = 0;
#pragma unroll
  for (int i = 0; i < kSel / 64; ++i) {
    if (i < w) { s0 += sc.part[i]; e0 += sc.part2[i]; }
    all_s += sc.part[i];
    all_e += sc.part2[i];
  }
  __syncthreads();
  const uint64_t below = (1ull << lane) - 1;
  const int eq_in = min(eqb, left);  // kept equals that base counts already
#pragma unroll
  for (int e = 0; e < EPT; ++e) {
    const int rank = e0 + __popcll(eq[e] & below), pos = s0 + __popcll(sure[e] & below) + min(rank, left) - eq_in;
    const bool is_eq = (eq[e] >> lane) & 1;
    if (((sure[e] >> lane) & 1) || (is_eq && rank < left)) put(pos, turn_row<EPT>(c0, e));
    s0 += __popcll(sure[e]);
    e0 += __popcll(eq[e]);
  }
  base += all_s + min(eqb + all_e, left) - eq_in;
  eqb += all_e;
}

// Row r of the (sequence, kv head) at km / vm, copied to its place by threads c of the row's `per`.
template <typename V>
__device__ __forceinline__ void copy_row(const EvictArgs& a, int bh, long r, int j, int c) {
  const long b = bh / a.by_h, h = bh - b * a.H;
  V x{}, y{};
  if (j >= 0) {
    x = *reinterpret_cast<const V*>(a.k + b * a.k_sb + h * a.k_sh + j * a.k_st + c);
    y = *reinterpret_cast<const V*>(a.v + b * a.v_sb + h * a.v_sh + j * a.v_st + c);
  }
  *reinterpret_cast<V*>(a.ko + r * a.row_bytes + c) = x;
  *reinterpret_cast<V*>(a.vo + r * a.row_bytes + c) = y;
  if (c == 0) a.mo[r] = j >= 0 ? *reinterpret_cast<const float*>(a.mass + b * a.m_sb + h * a.m_sh + j * 4L) : 0.f;
}

// V: bytes a thread moves at once, void: no gather here.  EPT: keys a thread holds.
template <typename V, int EPT>
__global__ __launch_bounds__(kSel) void evict_select_kernel(EvictArgs a) {
  constexpr bool FUSE = !std::is_void<V>::value;
  __shared__ __align__(16) int hist[3][kBins];
  __shared__ SelectScratch sc;
  const int b = (int)blockIdx.x / a.by_h, h = blockIdx.x - b * a.H, tid = threadIdx.x;
  const float* m = reinterpret_cast<const float*>(a.mass + b * a.m_sb + h * a.m_sh);
  for (int i = tid; i < 3 * kBins; i += kSel) hist[0][i] = 0;
  uint32_t key[EPT];
#pragma unroll
  for (int e = 0; e < EPT; ++e) {
    const int i = turn_row<EPT>(0, e);
    key[e] = i < a.T ? weight_key(m[i]) : 0u;
  }
  const EvictSeq q = evict_seq(a, b);
  int32_t* index = a.index + (long)blockIdx.x * a.keep;
  if (h == 0 && tid == 0 && a.kept) a.kept[b] = q.kept;
  for (int i = q.kept + tid; i < a.keep; i += kSel) index[i] = -1;
  uint32_t thr = 0;
  int left = q.need;
  if (q.need > 0) {
    __syncthreads();
    for (int pass = 0; pass < 3; ++pass) {
      const int nb = pass_bins(pass), sh = pass_shift(pass), up = pass == 0 ? 0 : pass_shift(pass - 1);
#pragma unroll
      for (int e = 0; e < EPT; ++e) {
        const int i = turn_row<EPT>(0, e);
        if (i >= q.lo && i < q.hi && (pass == 0 || (key[e] >> up) == (thr >> up)))
          atomicAdd(&hist[pass][(key[e] >> sh) & (nb - 1)], 1);
      }
      __syncthreads();
      if (tid < 64) find_bin_wave(hist[pass], nb, left, sc);
      __syncthreads();
      thr |= (uint32_t)sc.bin << sh;
      left = sc.need;
    }
  }
  int base = 0, eqb = 0;
  place_rows(q, key, 0, q.n, thr, left, base, eqb, sc, [&](int pos, int i) { index[pos] = i; });
  if constexpr (FUSE) {
    __syncthreads();  // (the indices, written by this work-group, are read back by it)
    const int per = a.row_bytes / (int)sizeof(V);
    for (int i = tid; i < a.keep * per; i += kSel) {
      const int r = i / a.by_per;
      copy_row<V>(a, blockIdx.x, (long)blockIdx.x * a.keep + r, index[r], (i - r * per) * (int)sizeof(V));
    }
  }
}

// Launch `pass` of a long row: adds up the row's histograms of the launch
// before (pass 1..3), narrows the last kept key by them, and writes its part's
// next histogram (pass 0..2) or its rows' places (pass 3).
//   hist  [B H][3][parts][kBins]
//   above [B H][parts]   rows of a part known to lie above the last kept key
//   state [B H][3][2]    after each launch: the key's bits so far, places left
__global__ __launch_bounds__(kSel) void evict_part_kernel(EvictArgs a, int pass, int parts, int* hist, int* above,
                                                          int* state) {
  __shared__ int sh_hist[kBins];
  __shared__ SelectScratch sc;
  const int bh = (int)blockIdx.x / a.by_parts, pt = blockIdx.x - bh * parts, tid = threadIdx.x;
  const int b = bh / a.by_h, h = bh - b * a.H;
  const float* m = reinterpret_cast<const float*>(a.mass + b * a.m_sb + h * a.m_sh);
  const int i0 = part_start(a.T, pt, a.by_parts), t1 = part_start(a.T, pt + 1, a.by_parts);
  // a turn's weights; the first turn's are on their way before anything else is known
  float x[kEpt];
  auto load_turn = [&](int c0) {
#pragma unroll
    for (int e = 0; e < kEpt; ++e) {
      const int i = turn_row<kEpt>(c0, e);
      x[e] = i < t1 ? m[i] : 0.f;
    }
  };
  load_turn(i0);
  const EvictSeq q = evict_seq(a, b);
  const int i1 = min(t1, q.n);
  uint32_t thr = 0;
  int left = q.need, prev_above = 0, prev_eq = 0;
  if (q.need > 0 && pass > 0) {
    if (pass > 1) { thr = (uint32_t)state[6 * bh + 2 * pass - 2]; left = state[6 * bh + 2 * pass - 1]; }
    const int nb = pass_bins(pass - 1), b0 = nb - 1 - 2 * tid;
    const int* src = hist + ((long)bh * 3 + pass - 1) * parts * kBins;
    int2 all = make_int2(0, 0), prev = make_int2(0, 0), mine = make_int2(0, 0);  // bins b0, b0 - 1
    if (b0 > 0)
      for (int p0 = 0; p0 < parts; p0 += 8) {  // eight parts' loads in flight
        int2 c[8];
#pragma unroll
        for (int u = 0; u < 8; ++u)  // (b0 is odd)
          c[u] = *reinterpret_cast<const int2*>(src + (long)min(p0 + u, parts - 1) * kBins + b0 - 1);
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int p = p0 + u;
          if (p < parts) { all.x += c[u].y; all.y += c[u].x; }
          if (p < pt) { prev.x += c[u].y; prev.y += c[u].x; }
          if (p == pt) mine = make_int2(c[u].y, c[u].x);
        }
      }
    int bin;
    find_bin(all.x, all.y, nb, left, bin, left, sc);
    thr |= (uint32_t)bin << pass_shift(pass - 1);
    // rows of the bins above it: this part's so far, and after the last pass those of the parts before
    const int2 use = pass == 3 ? prev : mine;
    int up = (b0 > bin ? use.x : 0) + (b0 - 1 > bin ? use.y : 0);
    int eq = (b0 == bin ? use.x : 0) + (b0 - 1 == bin ? use.y : 0);
    int tu, te;
    if (pass == 3 && tid < pt) up += above[(long)bh * parts + tid];  // (what the launches before found of them)
    block_scan2(up, eq, tu, te, sc);
    if (pass < 3) {
      if (tid == 0) {
        int* dst = above + (long)bh * parts + pt;
        *dst = (pass == 1 ? 0 : *dst) + tu;
      }
    } else {
      prev_above = tu;
      prev_eq = te;
    }
  }
  if (pass < 3) {
    if (q.need <= 0) return;
    if (pass > 0 && pt == 0 && tid == 0) { state[6 * bh + 2 * pass] = (int)thr; state[6 * bh + 2 * pass + 1] = left; }
    const int nb = pass_bins(pass), sh = pass_shift(pass), up = pass == 0 ? 0 : pass_shift(pass - 1);
    sh_hist[tid] = 0;
    sh_hist[tid + kSel] = 0;
    __syncthreads();
    for (int c0 = i0; c0 < i1; c0 += kChunk) {
      if (c0 > i0) load_turn(c0);
#pragma unroll
      for (int e = 0; e < kEpt; ++e) {
        const int i = turn_row<kEpt>(c0, e);
        const uint32_t key = weight_key(x[e]);
        if (i >= q.lo && i < min(i1, q.hi) && (pass == 0 || (key >> up) == (thr >> up)))
          atomicAdd(&sh_hist[(key >> sh) & (nb - 1)], 1);
      }
    }
    __syncthreads();
    int* dst = hist + (((long)bh * 3 + pass) * parts + pt) * kBins;
    dst[tid] = sh_hist[tid];
    dst[tid + kSel] = sh_hist[tid + kSel];
    return;
  }
  int32_t* index = a.index + (long)bh * a.keep;
  if (pt == 0) {
    if (h == 0 && tid == 0 && a.kept) a.kept[b] = q.kept;
    for (int i = q.kept + tid; i < a.keep; i += kSel) index[i] = -1;
  }
  // places taken by the parts before: rows kept for certain, above the last kept key, the first of its equals
  int base = min(i0, q.lo) + max(0, min(i0, q.n) - q.hi) + prev_above + min(prev_eq, left), eqb = prev_eq;
  for (int c0 = i0; c0 < i1; c0 += kChunk) {
    if (c0 > i0) load_turn(c0);
    uint32_t key[kEpt];
#pragma unroll
    for (int e = 0; e < kEpt; ++e) key[e] = weight_key(x[e]);
    place_rows(q, key, c0, i1, thr, left, base, eqb, sc, [&](int pos, int i) { index[pos] = i; });
  }
}

// One kept row a group of threads; V: bytes a thread moves at once.
template <typename V>
__global__ __launch_bounds__(256) void evict_gather_kernel(EvictArgs a, long n, int per) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const uint32_t r = (uint32_t)i / (uint32_t)per;  // (sequence, kv head, kept row); n is below 2^32
  copy_row<V>(a, (int)(r / (uint32_t)a.keep), r, a.index[r], (int)(i - (long)r * per) * (int)sizeof(V));
}

namespace {
int evict_parts(const carekv_evict_params& p) {
  if (p.n_keys <= 2 * kChunk) return 1;
  return (int)std::min((long)kMaxParts, ((long)p.n_keys + kChunk - 1) / kChunk);
}
long evict_ws(const carekv_evict_params& p) {
  const long parts = evict_parts(p);
  return parts == 1 ? 0 : (long)p.batch * p.n_kv_heads * (3 * parts * kBins + parts + 6) * 4;
}
int check_evict(const carekv_evict_params* pp) {
  CAREKV_REQUIRE(pp, "null argument");
  const carekv_evict_params& p = *pp;
  CAREKV_REQUIRE(p.batch >= 0 && p.n_kv_heads >= 0 && p.n_keys >= 0, "negative counts");
  CAREKV_REQUIRE(p.keep > 0 && p.sink >= 0 && p.recent >= 0 && (long)p.sink + p.recent <= p.keep,
                 "keep must be positive, sink and recent not negative and at most keep together");
  CAREKV_REQUIRE(p.n_keys < (1 << 30), "n_keys must be below 2^30");
  CAREKV_REQUIRE(p.row_bytes > 0 && p.row_bytes % 4 == 0, "rows must be a multiple of 4 bytes");
  CAREKV_REQUIRE(grid_fits((long)p.batch * p.n_kv_heads * evict_parts(p), kSel), "too many (sequence, kv head) rows");
  return CAREKV_OK;
}
}  // namespace

}  // namespace carekv

using namespace carekv;

extern "C" int64_t carekv_evict_rows_workspace_bytes(const carekv_evict_params* pp) {
  if (check_evict(pp) != CAREKV_OK) return -1;
  return evict_ws(*pp);
}

extern "C" int carekv_evict_rows(const carekv_evict_params* pp, const float* mass, const void* k, const void* v,
                                 const int32_t* lengths, void* k_out, void* v_out, float* mass_out, int32_t* index,
                                 int32_t* kept, void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = check_evict(pp);
  if (rc != CAREKV_OK) return rc;
  const carekv_evict_params& p = *pp;
  const long bh = (long)p.batch * p.n_kv_heads;
  if (bh == 0) return CAREKV_OK;
  const int parts = evict_parts(p);
  CAREKV_REQUIRE((p.n_keys == 0 || (mass && k && v)) && k_out && v_out && mass_out && index && (workspace || parts == 1),
                 "null argument");
  if (workspace_bytes < evict_ws(p)) {
    set_error("carekv_evict_rows: workspace too small (%lld < %lld)", (long long)workspace_bytes, (long long)evict_ws(p));
    return CAREKV_ESPACE;
  }
  EvictArgs a{};
  a.mass = (const char*)mass; a.k = (const char*)k; a.v = (const char*)v; a.lengths = lengths;
  a.ko = (char*)k_out; a.vo = (char*)v_out; a.mo = mass_out; a.index = index; a.kept = kept;
  a.m_sb = p.mass_sb * 4; a.m_sh = p.mass_sh * 4;
  a.k_sb = p.k_sb; a.k_sh = p.k_sh; a.k_st = p.k_st; a.v_sb = p.v_sb; a.v_sh = p.v_sh; a.v_st = p.v_st;
  a.H = p.n_kv_heads; a.T = p.n_keys; a.keep = p.keep; a.sink = p.sink; a.recent = p.recent; a.row_bytes = p.row_bytes;
  const uintptr_t bits = operand_bits(k, {{p.batch, p.k_sb}, {p.n_kv_heads, p.k_sh}, {p.n_keys, p.k_st}}) |
                         operand_bits(v, {{p.batch, p.v_sb}, {p.n_kv_heads, p.v_sh}, {p.n_keys, p.v_st}}) |
                         (uintptr_t)k_out | (uintptr_t)v_out | (uintptr_t)p.row_bytes;
  CAREKV_REQUIRE((bits & 3) == 0, "K and V rows must be 4-byte aligned");
  CAREKV_REQUIRE(parts == 1 || ((uintptr_t)workspace & 7) == 0, "the workspace must be 8-byte aligned");
  const bool wide = (bits & 15) == 0;
  const int per = p.row_bytes / (wide ? 16 : 4);
  const long n = bh * p.keep * per;
  a.by_h = FastDiv(p.n_kv_heads); a.by_parts = FastDiv(parts); a.by_per = FastDiv(per);
  CAREKV_REQUIRE(grid_fits((n + 255) / 256, 256), "too many kept rows");
  hipStream_t s = (hipStream_t)stream;
  if (parts == 1) {
    const bool fuse = (long)p.keep * p.row_bytes <= kFuseBytes;
    auto select = [&](auto ept) {
      constexpr int EPT = decltype(ept)::value;
      const dim3 grid((unsigned)bh), block(kSel);
      if (!fuse) hipLaunchKernelGGL((evict_select_kernel<void, EPT>), grid, block, 0, s, a);
      else if (wide) hipLaunchKernelGGL((evict_select_kernel<uint4, EPT>), grid, block, 0, s, a);
      else hipLaunchKernelGGL((evict_select_kernel<uint32_t, EPT>), grid, block, 0, s, a);
    };
    if (p.n_keys <= kChunk) select(std::integral_constant<int, kEpt>{});
    else select(std::integral_constant<int, 2 * kEpt>{});
    CAREKV_CHECK_LAUNCH("evict_select");
    if (fuse) return CAREKV_OK;
  } else {
    int* hist = (int*)workspace;
    int* above = hist + bh * 3 * parts * kBins;
    int* state = above + bh * parts;
    for (int pass = 0; pass < 4; ++pass) {
      hipLaunchKernelGGL(evict_part_kernel, dim3((unsigned)(bh * parts)), dim3(kSel), 0, s, a, pass, parts, hist, above,
                         state);
      CAREKV_CHECK_LAUNCH("evict_part");
    }
  }
  const dim3 grid((unsigned)((n + 255) / 256));
  if (wide) hipLaunchKernelGGL(evict_gather_kernel<uint4>, grid, dim3(256), 0, s, a, n, per);
  else hipLaunchKernelGGL(evict_gather_kernel<uint32_t>, grid, dim3(256), 0, s, a, n, per);
  CAREKV_CHECK_LAUNCH("evict_gather");
  return CAREKV_OK;
}
