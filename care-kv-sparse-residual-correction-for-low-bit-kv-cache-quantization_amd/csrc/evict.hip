// Rows of a K/V prompt kept by weight (evict_rows): per (sequence, kv head)
// the first `sink` and last `recent` rows, then the rows of largest weight
// (equal weights: the lower index), `keep` in all, in index order; their K, V
// and weight rows gathered.
//
// evict_select_kernel: one work-group a row.  Weights are mapped to unsigned
// keys of the same order (NaN to 0, below -inf); three passes of 11, 11 and 10
// bits of histograms in LDS find the key of the last kept row and how many of
// its equals are kept, a fourth pass counts in index order and writes the
// indices.  evict_gather_kernel copies the rows.
//
// Bound by memory: each weight and kept row read once, each kept row written.
#include "common.h"
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
};

// unsigned order of a weight: -inf < finite < +inf as unsigned integers, NaN lowest
__device__ __forceinline__ uint32_t weight_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);  // (-0 counts as +0)
  if (x != x) return 0u;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSel = 1024;  // threads of a select work-group

__global__ __launch_bounds__(kSel) void evict_select_kernel(EvictArgs a) {
  __shared__ int hist[2048];
  __shared__ int part[kSel / 64], s_bin, s_need;
  const int b = blockIdx.x / a.H, h = blockIdx.x % a.H, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const float* m = reinterpret_cast<const float*>(a.mass + b * a.m_sb + h * a.m_sh);
  const int n = a.lengths ? min(max(a.lengths[b], 0), a.T) : a.T;
  const int kept = min(n, a.keep);
  int32_t* index = a.index + (long)blockIdx.x * a.keep;
  if (h == 0 && tid == 0 && a.kept) a.kept[b] = kept;
  for (int i = kept + tid; i < a.keep; i += kSel) index[i] = -1;
  if (n <= a.keep) {
    for (int i = tid; i < n; i += kSel) index[i] = i;
    return;
  }
  // rows [lo, hi) compete for `need` places (1 <= need < hi - lo unless none is left); the others are kept
  const int lo = min(a.sink, n), hi = max(n - a.recent, lo);
  int need = kept - lo - (n - hi);
  uint32_t prefix = 0;  // bits found so far of the last kept row's key
  if (need > 0) {
    const int width[3] = {11, 11, 10};
    int sh = 32;
    for (int pass = 0; pass < 3; ++pass) {
      const int nb = 1 << width[pass], top = sh;
      sh -= width[pass];
      for (int i = tid; i < 2048; i += kSel) hist[i] = 0;
      __syncthreads();
      for (int i = lo + tid; i < hi; i += kSel) {
        const uint32_t key = weight_key(m[i]);
        if (pass == 0 || (key >> top) == (prefix >> top)) atomicAdd(&hist[(key >> sh) & (nb - 1)], 1);
      }
      __syncthreads();
      // the bin, from the top, where the count passes `need`: thread t has bins nb-1-2t, nb-2-2t
      const int b0 = nb - 1 - 2 * tid, c0 = 2 * tid < nb ? hist[b0] : 0, c1 = 2 * tid < nb ? hist[b0 - 1] : 0;
      int x = c0 + c1;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o, 64);
        if (lane >= o) x += y;
      }
      if (lane == 63) part[w] = x;
      __syncthreads();
      int before = x - c0 - c1;
      for (int i = 0; i < w; ++i) before += part[i];
      if (before < need && need <= before + c0 + c1) {
        const bool second = need > before + c0;
        s_bin = second ? b0 - 1 : b0;
        s_need = need - before - (second ? c0 : 0);
      }
      __syncthreads();
      prefix |= (uint32_t)s_bin << sh;
      need = s_need;
      __syncthreads();
    }
  }
  // kept: key > prefix, or one of the first `need` equals; in index order
  const bool any = kept - lo - (n - hi) > 0;
  int base = 0, eq_base = 0;
  for (int t0 = 0; t0 < n; t0 += kSel) {
    const int i = t0 + tid;
    bool sure = false, eq = false;
    if (i < n) {
      if (i < lo || i >= hi) {
        sure = true;
      } else if (any) {
        const uint32_t key = weight_key(m[i]);
        sure = key > prefix;
        eq = key == prefix;
      }
    }
    const uint64_t bs = __ballot(sure), be = __ballot(eq), below = (1ull << lane) - 1;
    if (lane == 0) part[w] = __popcll(bs) | (__popcll(be) << 16);
    __syncthreads();
    int ps = 0, pe = 0, ts = 0, te = 0;
    for (int j = 0; j < kSel / 64; ++j) {
      const int c = part[j];
      if (j < w) { ps += c & 0xffff; pe += c >> 16; }
      ts += c & 0xffff;
      te += c >> 16;
    }
    // equals before this thread's element, and how many of them are kept
    const int ebefore = eq_base + pe + __popcll(be & below);
    const int pos = base + ps + __popcll(bs & below) + min(ebefore, need) - min(eq_base, need);
    if (sure || (eq && ebefore < need)) index[pos] = i;
    base += ts + min(eq_base + te, need) - min(eq_base, need);
    eq_base += te;
    __syncthreads();
  }
}

// One kept row a group of threads; V: bytes a thread moves at once.
template <typename V>
__global__ __launch_bounds__(256) void evict_gather_kernel(EvictArgs a, long n, int per) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const long r = i / per;  // (sequence, kv head, kept row)
  const int c = (int)(i - r * per) * (int)sizeof(V);
  const long bh = r / a.keep, b = bh / a.H, h = bh - b * a.H;
  const int j = a.index[r];
  V x{}, y{};
  if (j >= 0) {
    x = *reinterpret_cast<const V*>(a.k + b * a.k_sb + h * a.k_sh + j * a.k_st + c);
    y = *reinterpret_cast<const V*>(a.v + b * a.v_sb + h * a.v_sh + j * a.v_st + c);
  }
  *reinterpret_cast<V*>(a.ko + r * a.row_bytes + c) = x;
  *reinterpret_cast<V*>(a.vo + r * a.row_bytes + c) = y;
  if (c == 0) a.mo[r] = j >= 0 ? *reinterpret_cast<const float*>(a.mass + b * a.m_sb + h * a.m_sh + j * 4L) : 0.f;
}

}  // namespace carekv

using namespace carekv;

extern "C" int carekv_evict_rows(const carekv_evict_params* pp, const float* mass, const void* k, const void* v,
                                 const int32_t* lengths, void* k_out, void* v_out, float* mass_out, int32_t* index,
                                 int32_t* kept, void* stream) {
  CAREKV_REQUIRE(pp, "null argument");
  const carekv_evict_params& p = *pp;
  CAREKV_REQUIRE(p.batch >= 0 && p.n_kv_heads >= 0 && p.n_keys >= 0, "negative counts");
  CAREKV_REQUIRE(p.keep > 0 && p.sink >= 0 && p.recent >= 0 && (long)p.sink + p.recent <= p.keep,
                 "keep must be positive, sink and recent not negative and at most keep together");
  CAREKV_REQUIRE(p.n_keys < (1 << 30), "n_keys must be below 2^30");
  CAREKV_REQUIRE(p.row_bytes > 0 && p.row_bytes % 4 == 0, "rows must be a multiple of 4 bytes");
  const long bh = (long)p.batch * p.n_kv_heads;
  if (bh == 0) return CAREKV_OK;
  CAREKV_REQUIRE((p.n_keys == 0 || (mass && k && v)) && k_out && v_out && mass_out && index, "null argument");
  CAREKV_REQUIRE(bh < (1L << 31), "too many (sequence, kv head) rows");
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
  const bool wide = (bits & 15) == 0;
  const int per = p.row_bytes / (wide ? 16 : 4);
  const long n = bh * p.keep * per;
  CAREKV_REQUIRE((n + 255) / 256 < (1L << 31), "too many kept rows");
  hipStream_t s = (hipStream_t)stream;
  hipLaunchKernelGGL(evict_select_kernel, dim3((unsigned)bh), dim3(kSel), 0, s, a);
  CAREKV_CHECK_LAUNCH("evict_select");
  const dim3 grid((unsigned)((n + 255) / 256));
  if (wide) hipLaunchKernelGGL(evict_gather_kernel<uint4>, grid, dim3(256), 0, s, a, n, per);
  else hipLaunchKernelGGL(evict_gather_kernel<uint32_t>, grid, dim3(256), 0, s, a, n, per);
  CAREKV_CHECK_LAUNCH("evict_gather");
  return CAREKV_OK;
}
