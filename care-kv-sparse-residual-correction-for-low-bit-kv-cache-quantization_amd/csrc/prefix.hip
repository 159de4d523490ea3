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
// and their sum is not.  The keys are split over work-groups until the GPU is
// full; prefix_join_kernel then joins the splits' (maximum, sum, O), kept in
// 32 bits, and the row's own part.
#include <algorithm>

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
  float* pml;            // [nsplit][rows][2] maximum (base 2), sum
  float* po;             // [nsplit][rows][D]
  long q_sb, q_sh, q_st, k_sh, k_st, v_sh, v_st, o_sb, o_sh, o_st, w_sb, w_sh, w_st;  // bytes
  long rows;             // n_kv_heads * M
  int B, Hq, Hkv, G, T, P, M, nqb, nsplit;
  float sm_log2;
};

// Row r of kv head hk: sequence, query head, query token.
struct PrefixRow {
  int b, h, t;
};
__device__ __forceinline__ PrefixRow prefix_row(const PrefixArgs& a, int hk, int r) {
  PrefixRow x;
  const int bg = r / a.T;
  x.t = r - bg * a.T;
  x.b = bg / a.G;
  x.h = hk * a.G + bg - x.b * a.G;
  return x;
}

template <typename ET, int D>
__global__ __launch_bounds__(256, 3) void prefix_attn_kernel(PrefixArgs a) {
  using V8 = typename ET::V8;
  using E = typename ET::E;
  constexpr int KT = 32, TT = KT / 16, NQ = 2, QW = 16 * NQ, QB = 4 * QW;
  constexpr int KRS = 2 * D + 16, VRS = 2 * D + 32;  // padded LDS rows: every bank once per read pattern
  constexpr int KS = D / 32, DT = D / 16, CHR = D / 8, NCH = 2 * KT * CHR / 256;
  constexpr int KBUF = KT * KRS, BUF = KBUF + KT * VRS;
  __shared__ __align__(16) char lds[2 * BUF];
  typedef short short4_t __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) short4_t lds_short4;

  // An XCD takes consecutive items, row blocks of one (head, split) next to
  // each other: they meet in its L2.
  const int n = gridDim.x;
  int it = blockIdx.x;
  if (n % 8 == 0) it = it % 8 * (n / 8) + it / 8;
  const int qblk = it % a.nqb, sp = it / a.nqb % a.nsplit, hk = it / a.nqb / a.nsplit;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c16 = lane & 15;
  const int r0 = qblk * QB + QW * w;  // first row of the wave
  const int tiles = (a.P + KT - 1) / KT;
  const int tile0 = (int)((long)sp * tiles / a.nsplit), tile1 = (int)((long)(sp + 1) * tiles / a.nsplit);
  const int j0 = tile0 * KT, keys = min(tile1 * KT, a.P) - j0;  // the split's keys (at least one)
  const __amdgpu_buffer_rsrc_t rk = make_rsrc(a.k + hk * a.k_sh + j0 * a.k_st, (uint32_t)((keys - 1) * a.k_st + 2 * D));
  const __amdgpu_buffer_rsrc_t rv = make_rsrc(a.v + hk * a.v_sh + j0 * a.v_st, (uint32_t)((keys - 1) * a.v_st + 2 * D));

  // Q^T operands: sub-block qb, step s -> row r0 + 16 qb + c16, dims 32s + 8g ..
  V8 qf[NQ][KS];
#pragma unroll
  for (int qb = 0; qb < NQ; ++qb) {
    const PrefixRow x = prefix_row(a, hk, min(r0 + 16 * qb + c16, a.M - 1));
    const char* qp = a.q + x.b * a.q_sb + x.h * a.q_sh + x.t * a.q_st;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const uint4 v = *reinterpret_cast<const uint4*>(qp + (32 * s + 8 * g) * 2);
      __builtin_memcpy(&qf[qb][s], &v, 16);
    }
  }

  uint32_t stg[NCH][4];
  auto load_tile = [&](int j) {
#pragma unroll
    for (int k = 0; k < NCH; ++k) {  // chunks k < NCH / 2 are K, the rest V
      const int rc = (threadIdx.x + 256 * k) % (KT * CHR), row = j * KT + rc / CHR, col = rc % CHR;
      // a row past the split reads zeros: its offset is at or past the resource's end
      const uint32_t st = (uint32_t)(k < NCH / 2 ? a.k_st : a.v_st);
      const uint32_t off = row < keys ? row * st + col * 16 : 0x7ffffff0u;
      const auto v = __builtin_amdgcn_raw_buffer_load_b128(k < NCH / 2 ? rk : rv, off, 0, 0);
      stg[k][0] = v[0]; stg[k][1] = v[1]; stg[k][2] = v[2]; stg[k][3] = v[3];
    }
  };
  auto store_tile = [&](int buf) {
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int rc = (threadIdx.x + 256 * k) % (KT * CHR), row = rc / CHR, col = rc % CHR;
      char* dst = lds + buf * BUF + (k < NCH / 2 ? row * KRS : KBUF + row * VRS) + col * 16;
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
  const float c = a.sm_log2;
  load_tile(0);
  store_tile(0);
  __syncthreads();
  if (nt > 1) load_tile(1);
  for (int j = 0; j < nt; ++j) {
    const char* kb = lds + (j & 1) * BUF;
    const char* vb = kb + KBUF;
    if (r0 < a.M) {
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
      // base-2 logits (a negative scale would turn a maximum of s into a minimum: scaled first)
#pragma unroll
      for (int tt = 0; tt < TT; ++tt)
#pragma unroll
        for (int qb = 0; qb < NQ; ++qb) s[tt][qb] *= c;
      if ((j + 1) * KT > keys) {  // the split's last tile: key 16 tt + 4g + i
        const int lim = keys - j * KT - 4 * g;
#pragma unroll
        for (int tt = 0; tt < TT; ++tt)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (16 * tt + i >= lim)
#pragma unroll
              for (int qb = 0; qb < NQ; ++qb) s[tt][qb][i] = -INFINITY;
      }
      V8 bp[NQ];
#pragma unroll
      for (int qb = 0; qb < NQ; ++qb) {
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) mx = fmaxf(mx, s[i / 4][qb][i % 4]);
        if (__any(mx > m_run[qb])) {  // columns that keep their maximum get a factor of exactly 1
          const float m_new = fmaxf(m_run[qb], col_max(mx));
          const float f = __builtin_amdgcn_exp2f(m_run[qb] - m_new);
          m_run[qb] = m_new;
          l_run[qb] *= f;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) o[qb][dt] *= f;
        }
        float ls = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float p = __builtin_amdgcn_exp2f(s[i / 4][qb][i % 4] - m_run[qb]);
          ls += p;
          bp[qb][i] = (E)p;
        }
        l_run[qb] += ls;
      }
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
    if (j + 1 < nt) store_tile((j + 1) & 1);
    if (j + 2 < nt) load_tile(j + 2);
    __syncthreads();
  }
  // the split's partial (lane: row r0 + 16qb + c16, dims 16dt + 4g ..)
#pragma unroll
  for (int qb = 0; qb < NQ; ++qb) {
    const float lt = col_sum(l_run[qb]);
    const int r = r0 + 16 * qb + c16;
    if (r < a.M) {
      const long pr = (long)sp * a.rows + (long)hk * a.M + r;
      float* dst = a.po + pr * D + 4 * g;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<float4_t*>(dst + 16 * dt) = o[qb][dt];
      if (g == 0) {
        a.pml[2 * pr] = m_run[qb];
        a.pml[2 * pr + 1] = lt;
      }
    }
  }
}

// Four dims of one row: the splits' partials and the row's own part joined in
// 32 bits.  A row that sees nothing (no prefix, lse_own = -inf) is zero with a
// log-sum-exp of -inf, whatever its own output holds.
template <typename ET>
__global__ __launch_bounds__(256) void prefix_join_kernel(PrefixArgs a, int D) {
  using E = typename ET::E;
  const int D4 = D / 4;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.rows * D4) return;
  const long pr = i / D4;
  const int d = (int)(i - pr * D4) * 4;
  const int hk = (int)(pr / a.M);
  const PrefixRow x = prefix_row(a, hk, (int)(pr - (long)hk * a.M));
  const long lrow = ((long)x.b * a.Hq + x.h) * a.T + x.t;
  const float lo = a.own ? a.own_lse[lrow] * kLog2e : -INFINITY;
  float m = lo;
  for (int s = 0; s < a.nsplit; ++s) m = fmaxf(m, a.pml[2 * (s * a.rows + pr)]);
  float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
  float L = 0.f;
  if (lo != -INFINITY) {  // (NaN goes on as NaN)
    const float f = __builtin_amdgcn_exp2f(lo - m);
    const E* p = reinterpret_cast<const E*>(a.own + x.b * a.w_sb + x.h * a.w_sh + x.t * a.w_st) + d;
    O = make_float4(f * (float)p[0], f * (float)p[1], f * (float)p[2], f * (float)p[3]);
    L = f;
  }
  for (int s = 0; s < a.nsplit; ++s) {
    const long r = s * a.rows + pr;
    const float f = __builtin_amdgcn_exp2f(a.pml[2 * r] - m);
    const float4 v = *reinterpret_cast<const float4*>(a.po + r * D + d);
    L = fmaf(f, a.pml[2 * r + 1], L);
    O.x = fmaf(f, v.x, O.x); O.y = fmaf(f, v.y, O.y); O.z = fmaf(f, v.z, O.z); O.w = fmaf(f, v.w, O.w);
  }
  const bool none = L == 0.f;
  const float inv = none ? 0.f : 1.f / L;
  E* dst = reinterpret_cast<E*>(a.out + x.b * a.o_sb + x.h * a.o_sh + x.t * a.o_st) + d;
  dst[0] = (E)(O.x * inv); dst[1] = (E)(O.y * inv); dst[2] = (E)(O.z * inv); dst[3] = (E)(O.w * inv);
  if (a.lse && d == 0) a.lse[lrow] = none ? -INFINITY : (m + __log2f(L)) * kLn2;
}

namespace {
// Splits of the keys: until 768 work-groups (3 a CU) are there, each of at
// least 4 tiles, and no split's rows past 2^30 bytes (32-bit offsets).
int prefix_splits(const carekv_prefix_params& p) {
  const long M = (long)p.batch * p.seq_len * (p.n_heads / p.n_kv_heads);
  const long wgs = (M + 127) / 128 * p.n_kv_heads, tiles = ((long)p.prefix_len + 31) / 32;
  if (tiles == 0 || wgs == 0) return 0;
  long s = std::max(1L, std::min(768 / wgs, (tiles + 3) / 4));
  const long st = p.prefix_len > 1 ? 2 * std::max(p.k_st, p.v_st) : 0;
  while (s < tiles && ((tiles + s - 1) / s + 1) * 32 * st >= (1L << 30)) ++s;
  return (int)std::min(s, tiles);
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
  return ns * rows * (2 + p.head_dim) * 4;
}
}  // namespace

}  // namespace carekv

using namespace carekv;

extern "C" int64_t carekv_prefix_attn_workspace_bytes(const carekv_prefix_params* pp) {
  if (check_prefix(pp) != CAREKV_OK) return -1;
  return prefix_ws(*pp, prefix_splits(*pp));
}

extern "C" int carekv_prefix_attn(const carekv_prefix_params* pp, const void* q, const void* k, const void* v,
                                  const void* own, const float* own_lse, void* out, float* lse, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  const int rc = check_prefix(pp);
  if (rc != CAREKV_OK) return rc;
  const carekv_prefix_params& p = *pp;
  const long rows = (long)p.batch * p.seq_len * p.n_heads;
  if (rows == 0) return CAREKV_OK;
  CAREKV_REQUIRE(q && out && (workspace || prefix_splits(p) == 0) && (p.prefix_len == 0 || (k && v)) && !own == !own_lse, "null argument");
  const uintptr_t bits = operand_bits(q, {{p.batch, 2 * p.q_sb}, {p.n_heads, 2 * p.q_sh}, {p.seq_len, 2 * p.q_st}}) |
                         operand_bits(k, {{p.n_kv_heads, 2 * p.k_sh}, {p.prefix_len, 2 * p.k_st}}) |
                         operand_bits(v, {{p.n_kv_heads, 2 * p.v_sh}, {p.prefix_len, 2 * p.v_st}}) |
                         (uintptr_t)workspace;
  CAREKV_REQUIRE((bits & 15) == 0, "q, k and v rows must be 16-byte aligned");
  const int ns = prefix_splits(p);
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
  a.P = p.prefix_len; a.M = p.batch * a.G * p.seq_len; a.rows = rows; a.nqb = (a.M + 127) / 128; a.nsplit = ns;
  a.po = (float*)workspace;
  a.pml = a.po + ns * rows * p.head_dim;
  a.sm_log2 = (float)((double)p.sm_scale * 1.4426950408889634074);
  hipStream_t s = (hipStream_t)stream;
  const long wgs = (long)a.nqb * a.Hkv * ns, jt = rows * (p.head_dim / 4);
  CAREKV_REQUIRE(wgs < (1L << 31), "too many row blocks");
  return dispatch_elem_d(p.dtype, p.head_dim, [&](auto et, auto d) {
    using ET = decltype(et);
    if (ns > 0) {
      hipLaunchKernelGGL((prefix_attn_kernel<ET, decltype(d)::value>), dim3((unsigned)wgs), dim3(256), 0, s, a);
      CAREKV_CHECK_LAUNCH("prefix_attn");
    }
    hipLaunchKernelGGL((prefix_join_kernel<ET>), dim3((unsigned)((jt + 255) / 256)), dim3(256), 0, s, a, p.head_dim);
    CAREKV_CHECK_LAUNCH("prefix_join");
    return CAREKV_OK;
  });
}
