// Attention weight that each key has gathered (attention_mass):
//   mass[b][g][j] = sum over the query heads h of kv head g and the query rows
//   i that see key j of e^(scale q_i . k_j - lse_i)
// with lse_i the log-sum-exp of row i's visible scores, given or computed here.
// Query row i stands at position q_start + i and sees the keys j below
// min(length, position + 1) (not causal: below the length).
//
// Key-stationary: a work-group keeps 128 keys (4 waves of 32, the A operand of
// S^T = K Q^T in registers) and walks over 32-query tiles of every head of the
// group staged in LDS, so that a key's weights add up in one lane group's
// registers and nothing of size queries x keys is written.  Rows are walked a
// head at a time from the first that sees the block, or, where a head has
// fewer rows than a tile, all heads' rows as one list.  Without lse a first
// pass of the same walk writes each block's (maximum, sum) per row and
// mass_join_kernel joins them; the second pass reads K again from the caches.
//
// Sums: a lane adds at most kFlush tiles' weights before they go to an outer
// sum, so that a key's total over 2^15 rows keeps the accuracy of a short sum.
// The rows' statistics are (M, w): a weight is 2^(x - M) w, with w = 1 / sum,
// or for a given lse the part of lse log2(e) that a 32-bit M does not hold.
#include <algorithm>

#include "mfma16.h"

namespace carekv {

struct MassArgs {
  const char* q;
  const char* k;
  const float* lse;        // [B][Hq][Tq], or null
  const int32_t* q_start;  // [B], or null: the last Tq of the length
  const int32_t* lengths;  // [B], or null
  float* out;
  float* part;             // [B][Hkv][rows][nkb][2] maximum (base 2), sum
  float* stat;             // [B][Hkv][rows][2] M, w
  long q_sb, q_sh, q_st, k_sb, k_sh, k_st;  // bytes
  long o_sb, o_sh;                          // elements
  int B, Hq, Hkv, G, Tq, Tk, nkb, causal, accumulate;
  int nseg, seg;           // the walk: nseg lists of seg rows
  float sm_log2;
};

constexpr int kMassKeys = 128, kMassTile = 32, kFlush = 16;

// Keys that row (head-local) t of sequence b sees: j < the result (0: none)
__device__ __forceinline__ int mass_limit(const MassArgs& a, int b, int t) {
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.Tk) : a.Tk;
  if (!a.causal) return len;
  const long pos = (a.q_start ? (long)a.q_start[b] : (long)len - a.Tq) + t;
  return (int)max(0L, min((long)len, pos + 1));
}

template <typename ET, int D, bool STATS>
__global__ __launch_bounds__(256) void mass_kernel(MassArgs a) {
  using V8 = typename ET::V8;
  constexpr int KS = D / 32, QRS = 2 * D + 16, CHR = D / 8, NCH = kMassTile * CHR / 256;
  static_assert(NCH >= 1, "a thread stages whole chunks");
  __shared__ __align__(16) char lds[2][kMassTile * QRS];
  __shared__ float s_m[2][kMassTile], s_w[2][kMassTile];
  __shared__ int s_lim[2][kMassTile];
  __shared__ float s_red[STATS ? 4 * kMassTile * 2 : 1];
  const int hb = blockIdx.x % (a.Hkv * a.B), kb = blockIdx.x / (a.Hkv * a.B);
  const int b = hb / a.Hkv, hk = hb % a.Hkv;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c16 = lane & 15;
  const int j0 = kb * kMassKeys + 32 * w;  // first key of the wave
  // K operands: tokens j0 + 16 tt + c16, dims 32 s + 8 g .. (keys past the end: the last one, masked below)
  V8 kf[2][KS];
#pragma unroll
  for (int tt = 0; tt < 2; ++tt) {
    const char* kp = a.k + b * a.k_sb + hk * a.k_sh + (long)min(j0 + 16 * tt + c16, a.Tk - 1) * a.k_st;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const uint4 v = *reinterpret_cast<const uint4*>(kp + (32 * s + 8 * g) * 2);
      __builtin_memcpy(&kf[tt][s], &v, 16);
    }
  }
  const long rows = (long)a.G * a.Tq;
  const long hrow = (long)hb * rows;  // first row of this (sequence, kv head) in part / stat
  // rows of a list below t_first see nothing of the block
  int t_first = 0;
  if (a.causal && a.nseg > 1) {
    const int len = a.lengths ? min(max(a.lengths[b], 0), a.Tk) : a.Tk;
    const long qs = a.q_start ? (long)a.q_start[b] : (long)len - a.Tq;
    t_first = (int)min((long)a.seg, max(0L, (long)kb * kMassKeys - qs));
    if ((long)kb * kMassKeys >= len) t_first = a.seg;
  }
  const int per = (a.seg - t_first + kMassTile - 1) / kMassTile, nt = per * a.nseg;
  uint32_t stg[NCH][4];
  float n_m = 0.f, n_w = 0.f;
  int n_lim = 0;
  // row of list position p of list sg: head sg and row p, or the rows of all heads in order
  auto locate = [&](int j, int p, int& h, int& t) {
    const int sg = j / per, i = t_first + (j - sg * per) * kMassTile + p;
    if (a.nseg > 1) { h = sg; t = i; }
    else { h = i / a.Tq; t = i - h * a.Tq; }
    return i < a.seg;
  };
  auto load_tile = [&](int j) {
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int cid = threadIdx.x + 256 * k, row = cid / CHR, col = cid % CHR;
      int h, t;
      const bool in = locate(j, row, h, t);
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (in) v = *reinterpret_cast<const uint4*>(a.q + b * a.q_sb + ((long)hk * a.G + h) * a.q_sh + (long)t * a.q_st + col * 16);
      stg[k][0] = v.x; stg[k][1] = v.y; stg[k][2] = v.z; stg[k][3] = v.w;
    }
    if (threadIdx.x < kMassTile) {
      int h, t;
      const bool in = locate(j, threadIdx.x, h, t);
      n_lim = in ? mass_limit(a, b, t) : 0;
      if (!STATS && in) {
        const float2 st = *reinterpret_cast<const float2*>(a.stat + 2 * (hrow + (long)h * a.Tq + t));
        n_m = st.x; n_w = st.y;
      } else {
        n_m = 0.f; n_w = 0.f;
      }
    }
  };
  auto store_tile = [&](int buf) {
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int cid = threadIdx.x + 256 * k, row = cid / CHR, col = cid % CHR;
      *reinterpret_cast<uint4*>(lds[buf] + row * QRS + col * 16) = make_uint4(stg[k][0], stg[k][1], stg[k][2], stg[k][3]);
    }
    if (threadIdx.x < kMassTile) {
      s_lim[buf][threadIdx.x] = n_lim; s_m[buf][threadIdx.x] = n_m; s_w[buf][threadIdx.x] = n_w;
    }
  };
  float acc[8], sum[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = sum[i] = 0.f;
  if (nt > 0) {
    load_tile(0);
    store_tile(0);
  }
  __syncthreads();
  if (nt > 1) load_tile(1);
  for (int j = 0; j < nt; ++j) {
    const char* qb_ = lds[j & 1];
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) {
      float4_t s[2] = {float4_t{0.f, 0.f, 0.f, 0.f}, float4_t{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        V8 qf;
        *reinterpret_cast<uint4*>(&qf) = *reinterpret_cast<const uint4*>(qb_ + (16 * qb + c16) * QRS + (32 * ks + 8 * g) * 2);
        s[0] = ET::mfma(kf[0][ks], qf, s[0]);
        s[1] = ET::mfma(kf[1][ks], qf, s[1]);
      }
      const int col = 16 * qb + c16;
      const int lim = s_lim[j & 1][col] - j0 - 4 * g;  // token 16 tt + i of the lane is seen below it
      const bool edge = __any(lim < 32 - 4 * g);
      if (STATS) {
        float x[8], mx = kLowest;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] = s[i / 4][i % 4] * a.sm_log2;
          if (edge && 16 * (i / 4) + i % 4 >= lim) x[i] = -INFINITY;
          mx = fmaxf(mx, x[i]);
        }
        mx = col_max(mx);
        float l = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) l += __builtin_amdgcn_exp2f(x[i] - mx);
        l = col_sum(l);
        if (g == 0) {
          s_red[(w * kMassTile + col) * 2] = mx;
          s_red[(w * kMassTile + col) * 2 + 1] = l;
        }
      } else {
        const float m = s_m[j & 1][col], wt = s_w[j & 1][col];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float p = __builtin_amdgcn_exp2f(fmaf(s[i / 4][i % 4], a.sm_log2, -m));
          if (!edge) acc[i] = fmaf(p, wt, acc[i]);
          else if (16 * (i / 4) + i % 4 < lim) acc[i] = fmaf(p, wt, acc[i]);
        }
      }
    }
    if (!STATS && (j + 1) % kFlush == 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) { sum[i] += acc[i]; acc[i] = 0.f; }
    }
    if (j + 1 < nt) store_tile((j + 1) & 1);
    if (j + 2 < nt) load_tile(j + 2);
    __syncthreads();
    if (STATS) {
      if (threadIdx.x < kMassTile) {
        int h, t;
        if (locate(j, threadIdx.x, h, t)) {
          float m = kLowest, l = 0.f;
          for (int i = 0; i < 4; ++i) m = fmaxf(m, s_red[(i * kMassTile + threadIdx.x) * 2]);
          for (int i = 0; i < 4; ++i)
            l += s_red[(i * kMassTile + threadIdx.x) * 2 + 1] * __builtin_amdgcn_exp2f(s_red[(i * kMassTile + threadIdx.x) * 2] - m);
          float* p = a.part + 2 * ((hrow + (long)h * a.Tq + t) * a.nkb + kb);
          p[0] = m;
          p[1] = l;
        }
      }
      __syncthreads();
    }
  }
  if (!STATS) {
    // over the 16 query columns, in a fixed order
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v = sum[i] + acc[i];
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) v += __shfl_xor(v, o, 64);
      const int key = j0 + 16 * (i / 4) + 4 * g + i % 4;
      if (c16 == 0 && key < a.Tk) {
        float* p = a.out + b * a.o_sb + hk * a.o_sh + key;
        *p = a.accumulate ? *p + v : v;
      }
    }
  }
}

// (M, w) of every row: from the blocks' partials, or from the given lse.  A
// row that sees nothing, or whose lse is infinite, has (inf, 0): weights of 0.
__global__ __launch_bounds__(256) void mass_join_kernel(MassArgs a) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  const long per_b = (long)a.Hq * a.Tq;
  if (i >= a.B * per_b) return;
  const int b = (int)(i / per_b), t = (int)(i % a.Tq);
  float m = INFINITY, w = 0.f;
  if (a.lse) {
    // lse log2(e) = M + rest: M the rounded product, rest what it lost (NaN goes on as NaN)
    const float l = a.lse[i];
    if (!(fabsf(l) >= 1e30f)) {
      m = l * kLog2e;
      const float rest = fmaf(l, kLog2e, -m) + l * 1.9259629911266174e-8f;  // log2(e) - float(log2(e))
      w = __builtin_amdgcn_exp2f(-rest);
    }
  } else {
    // a causal row has partials of the blocks that it can see
    const int lim = mass_limit(a, b, t), nb = (lim + kMassKeys - 1) / kMassKeys;
    const float* p = a.part + 2 * i * a.nkb;
    float mx = kLowest, l = 0.f;
    for (int s = 0; s < nb; ++s) mx = fmaxf(mx, p[2 * s]);
    for (int s = 0; s < nb; ++s) l += p[2 * s + 1] * __builtin_amdgcn_exp2f(p[2 * s] - mx);
    if (l != 0.f) {
      m = mx;
      w = 1.f / l;
    }
  }
  a.stat[2 * i] = m;
  a.stat[2 * i + 1] = w;
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
  CAREKV_REQUIRE(p.n_keys < (1 << 30) && (long)p.n_queries * (p.n_heads / p.n_kv_heads) < (1L << 30),
                 "n_keys and the rows of a kv head must be below 2^30");
  CAREKV_REQUIRE((long)p.batch * p.n_kv_heads * ((p.n_keys + 127L) / 128) < (1L << 31), "too many key blocks");
  return CAREKV_OK;
}
long mass_ws(const carekv_mass_params& p, bool have_lse) {
  const long rows = (long)p.batch * p.n_heads * p.n_queries, nkb = (p.n_keys + kMassKeys - 1) / kMassKeys;
  return rows * 8 * (1 + (have_lse ? 0 : nkb)) + 256;
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
  CAREKV_REQUIRE(k && out && workspace && (p.n_queries == 0 || q), "null argument");
  uintptr_t bits = (uintptr_t)q | (uintptr_t)k | (uintptr_t)workspace;
  for (int64_t x : {p.q_sb, p.q_sh, p.q_st, p.k_sb, p.k_sh, p.k_st}) bits |= (uintptr_t)(2 * x);
  CAREKV_REQUIRE((bits & 15) == 0, "q and k rows must be 16-byte aligned");
  if (workspace_bytes < mass_ws(p, lse != nullptr)) {
    set_error("carekv_attention_mass: workspace too small (%lld < %lld)", (long long)workspace_bytes,
              (long long)mass_ws(p, lse != nullptr));
    return CAREKV_ESPACE;
  }
  MassArgs a{};
  a.q = (const char*)q; a.k = (const char*)k; a.lse = lse; a.q_start = q_start; a.lengths = lengths; a.out = out;
  a.q_sb = 2 * p.q_sb; a.q_sh = 2 * p.q_sh; a.q_st = 2 * p.q_st; a.k_sb = 2 * p.k_sb; a.k_sh = 2 * p.k_sh;
  a.k_st = 2 * p.k_st; a.o_sb = p.out_sb; a.o_sh = p.out_sh;
  a.B = p.batch; a.Hq = p.n_heads; a.Hkv = p.n_kv_heads; a.G = p.n_heads / p.n_kv_heads; a.Tq = p.n_queries;
  a.Tk = p.n_keys; a.nkb = (p.n_keys + kMassKeys - 1) / kMassKeys; a.causal = p.causal != 0;
  a.accumulate = p.accumulate != 0;
  if (p.n_queries >= kMassTile) { a.nseg = a.G; a.seg = a.Tq; }
  else { a.nseg = 1; a.seg = a.G * a.Tq; }
  a.sm_log2 = (float)((double)p.sm_scale * 1.4426950408889634074);
  const long rows = (long)p.batch * p.n_heads * p.n_queries;
  a.stat = (float*)workspace;
  a.part = a.stat + 2 * rows;
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)((long)a.B * a.Hkv * a.nkb));
  CAREKV_REQUIRE((rows + 255) / 256 < (1L << 31), "too many query rows");
  return dispatch_elem_d(p.dtype, p.head_dim, [&](auto et, auto d) {
    using ET = decltype(et);
    constexpr int D = decltype(d)::value;
    if (!lse && rows > 0) {
      hipLaunchKernelGGL((mass_kernel<ET, D, true>), grid, dim3(256), 0, s, a);
      CAREKV_CHECK_LAUNCH("mass (row statistics)");
    }
    if (rows > 0) {
      hipLaunchKernelGGL(mass_join_kernel, dim3((unsigned)((rows + 255) / 256)), dim3(256), 0, s, a);
      CAREKV_CHECK_LAUNCH("mass_join");
    }
    hipLaunchKernelGGL((mass_kernel<ET, D, false>), grid, dim3(256), 0, s, a);
    CAREKV_CHECK_LAUNCH("mass");
    return CAREKV_OK;
  });
}
