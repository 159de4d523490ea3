// Drafted tokens against the model's probabilities (verify_drafts): token x_t of
// a sequence is accepted while u_t q_t(x_t) < p_t(x_t), and behind the n accepted
// ones comes the smallest i with
//   w_0 + .. + w_i > u_next (w_0 + .. + w_(V-1)),
// w = max(p_n - q_n, 0) where a token was rejected (and any w is over 0), else
// p_n.  Products and sums are 64 bits: the order of their rounding moves a border
// between tokens by 2^-50 of the sum, in 32 bits by as much as a token holds.
//
// Bound by reading the one row of p and q that the next token is drawn from.  A
// row is cut over work-groups, which add up their parts; a second launch finds
// the part and the place in it.
#include <algorithm>

#include "common.h"
#include "host_util.h"

namespace carekv {

struct VerifyArgs {
  const char* p;         // [B][T + 1][V]
  const char* q;         // [B][T][V], or null: all of q_t is on x_t
  const int64_t* draft;  // [B][T]
  const float* u;        // [B][T]
  const float* u_next;   // [B]
  const int32_t* counts; // or null
  int32_t* tokens;       // [B][T + 1]
  int32_t* accepted;     // [B]
  double* sums;          // [B][parts][2]: of max(p - q, 0), of p
  long p_sb, p_st, q_sb, q_st, draft_sb, u_sb;  // elements
  int T, V, parts, step; // a part is step values
};

// How many of sequence b's tokens are accepted, by the work-group's first wave, to all of its threads.
template <typename E>
__device__ __forceinline__ int count_accepted(const VerifyArgs& a, int b, int count) {
  __shared__ int s_n;
  if (threadIdx.x < 64) {
    int n = 0;
    for (; n < count; n += 64) {
      const int t = n + threadIdx.x;
      bool ok = false;
      if (t < count) {
        const long x = a.draft[b * a.draft_sb + t];
        if (x >= 0 && x < a.V) {  // (any other token is rejected)
          const double px = (double)(float)reinterpret_cast<const E*>(a.p)[b * a.p_sb + t * a.p_st + x];
          const double qx = a.q ? (double)(float)reinterpret_cast<const E*>(a.q)[b * a.q_sb + t * a.q_st + x] : 1.0;
          ok = (double)a.u[b * a.u_sb + t] * qx < px;
        }
      }
      const unsigned long long m = __ballot(ok);
      if (m != ~0ull) {
        n += __ffsll((long long)~m) - 1;
        break;
      }
    }
    if (threadIdx.x == 0) s_n = min(n, count);
  }
  __syncthreads();
  return s_n;
}

// The weights of row n: max(p - q, 0) and p, 0 where they are not over 0.
template <typename E>
struct Weights {
  const E* p;
  const E* q;
  long x;      // the token whose weight is 0 where q is not given, -1: none
  bool rest;   // whether a token was rejected
  __device__ __forceinline__ Weights(const VerifyArgs& a, int b, int n, int count)
      : p(reinterpret_cast<const E*>(a.p) + b * a.p_sb + n * a.p_st), q(nullptr), x(-1), rest(n < count) {
    if (!rest) return;
    if (a.q) q = reinterpret_cast<const E*>(a.q) + b * a.q_sb + n * a.q_st;
    else x = a.draft[b * a.draft_sb + n];
  }
  __device__ __forceinline__ void at(int i, double& r, double& w) const {
    const double v = (double)(float)p[i], d = q ? v - (double)(float)q[i] : i == x ? 0.0 : v;
    w = v > 0.0 ? v : 0.0;
    r = rest ? (d > 0.0 ? d : 0.0) : w;
  }
};

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

template <typename E>
__global__ __launch_bounds__(256) void verify_sums_kernel(VerifyArgs a) {
  const int b = blockIdx.y;
  const int count = min(max(a.counts ? a.counts[b] : a.T, 0), a.T);
  const int n = count_accepted<E>(a, b, count);
  const Weights<E> w(a, b, n, count);
  const int i0 = blockIdx.x * a.step, i1 = min(i0 + a.step, a.V);
  double r = 0.0, s = 0.0;
  for (int i = i0 + threadIdx.x; i < i1; i += 256) {
    double x, y;
    w.at(i, x, y);
    r += x;
    s += y;
  }
  __shared__ double s_r[4], s_s[4];
  r = wave_sum_d(r);
  s = wave_sum_d(s);
  if ((threadIdx.x & 63) == 0) { s_r[threadIdx.x >> 6] = r; s_s[threadIdx.x >> 6] = s; }
  __syncthreads();
  if (threadIdx.x == 0) {
    double* dst = a.sums + 2 * ((long)b * a.parts + blockIdx.x);
    dst[0] = (s_r[0] + s_r[1]) + (s_r[2] + s_r[3]);
    dst[1] = (s_s[0] + s_s[1]) + (s_s[2] + s_s[3]);
  }
}

template <typename E>
__global__ __launch_bounds__(256) void verify_pick_kernel(VerifyArgs a) {
  const int b = blockIdx.x;
  const int count = min(max(a.counts ? a.counts[b] : a.T, 0), a.T);
  const int n = count_accepted<E>(a, b, count);
  const Weights<E> w(a, b, n, count);
  __shared__ double s_base, s_goal;
  __shared__ int s_part, s_kind;
  if (threadIdx.x == 0) {
    const double* sums = a.sums + 2 * (long)b * a.parts;
    double r = 0.0, s = 0.0;
    for (int i = 0; i < a.parts; ++i) { r += sums[2 * i]; s += sums[2 * i + 1]; }
    const int kind = r > 0.0 ? 0 : 1;
    const double total = kind ? s : r;
    // the first part whose end passes the goal; none does for u_next of 1 and more: the last with any weight
    double goal = (double)a.u_next[b] * total, base = 0.0, at = 0.0;
    if (!(goal >= 0.0)) goal = 0.0;
    int part = -1;
    for (int i = 0; i < a.parts; ++i) {
      const double x = sums[2 * i + kind];
      if (x > 0.0) {
        part = i;
        base = at;
        if (at + x > goal) break;
      }
      at += x;
    }
    s_base = base;
    s_goal = goal;
    s_part = total > 0.0 ? part : -1;
    s_kind = kind;
  }
  __syncthreads();
  const int part = s_part, kind = s_kind;
  int token = -1;
  if (part >= 0) {
    // a thread's run of the part, the runs' sums, and the place in the run that passes the goal
    const int i0 = part * a.step, i1 = min(i0 + a.step, a.V), run = (i1 - i0 + 255) / 256;
    const int j0 = min(i0 + (int)threadIdx.x * run, i1), j1 = min(j0 + run, i1);
    double mine = 0.0;
    for (int i = j0; i < j1; ++i) {
      double x[2];
      w.at(i, x[0], x[1]);
      mine += x[kind];
    }
    __shared__ double s_run[256];
    __shared__ int s_who;
    s_run[threadIdx.x] = mine;
    __syncthreads();
    if (threadIdx.x == 0) {
      double at = s_base;
      int who = 0;
      double base = at;
      for (int i = 0; i < 256; ++i) {
        if (s_run[i] > 0.0) {
          who = i;
          base = at;
          if (at + s_run[i] > s_goal) break;
        }
        at += s_run[i];
      }
      s_who = who;
      s_base = base;
    }
    __syncthreads();
    if ((int)threadIdx.x == s_who) {
      double at = s_base;
      for (int i = j0; i < j1; ++i) {
        double x[2];
        w.at(i, x[0], x[1]);
        at += x[kind];
        if (x[kind] > 0.0) {
          token = i;
          if (at > s_goal) break;
        }
      }
      s_part = token;
    }
    __syncthreads();
    token = s_part;
  }
  for (int t = threadIdx.x; t <= a.T; t += 256)
    a.tokens[(long)b * (a.T + 1) + t] = t < n ? (int32_t)a.draft[b * a.draft_sb + t] : t == n ? token : -1;
  if (threadIdx.x == 0) a.accepted[b] = n;
}

namespace {
// Parts of a row: until 1024 work-groups are there, of at least 2048 values each.
int verify_parts(const carekv_verify_params& p) {
  const long most = (p.vocab + 2047L) / 2048, want = std::max(1L, 1024L / std::max(p.batch, 1));
  return (int)std::max(1L, std::min(most, want));
}
int check_verify(const carekv_verify_params* pp) {
  CAREKV_REQUIRE(pp, "null argument");
  const carekv_verify_params& p = *pp;
  CAREKV_REQUIRE(p.dtype >= CAREKV_F16 && p.dtype <= CAREKV_F32, "dtype must be CAREKV_F16, CAREKV_BF16 or CAREKV_F32");
  CAREKV_REQUIRE(p.batch >= 0 && p.n_drafts >= 0 && p.vocab > 0, "negative counts, or no vocabulary");
  CAREKV_REQUIRE(p.batch < 65536 && p.n_drafts < (1 << 20) && p.vocab < (1 << 30), "too many sequences, drafts or tokens");
  return CAREKV_OK;
}
}  // namespace

}  // namespace carekv

using namespace carekv;

extern "C" int64_t carekv_verify_drafts_workspace_bytes(const carekv_verify_params* pp) {
  if (check_verify(pp) != CAREKV_OK) return -1;
  return 16L * pp->batch * verify_parts(*pp);
}

extern "C" int carekv_verify_drafts(const carekv_verify_params* pp, const int64_t* draft, const void* target_probs,
                                    const void* draft_probs, const float* u, const float* u_next,
                                    const int32_t* counts, int32_t* tokens, int32_t* accepted, void* workspace,
                                    int64_t workspace_bytes, void* stream) {
  const int rc = check_verify(pp);
  if (rc != CAREKV_OK) return rc;
  const carekv_verify_params& p = *pp;
  if (p.batch == 0) return CAREKV_OK;
  CAREKV_REQUIRE(target_probs && u_next && tokens && accepted && workspace && (p.n_drafts == 0 || (draft && u)), "null argument");
  VerifyArgs a{};
  a.p = (const char*)target_probs; a.q = p.n_drafts ? (const char*)draft_probs : nullptr; a.draft = draft; a.u = u;
  a.u_next = u_next; a.counts = counts; a.tokens = tokens; a.accepted = accepted; a.sums = (double*)workspace;
  a.p_sb = p.target_sb; a.p_st = p.target_st; a.q_sb = p.draft_probs_sb; a.q_st = p.draft_probs_st;
  a.draft_sb = p.draft_sb; a.u_sb = p.u_sb;
  a.T = p.n_drafts; a.V = p.vocab; a.parts = verify_parts(p);
  a.step = (p.vocab + a.parts - 1) / a.parts;
  a.parts = (p.vocab + a.step - 1) / a.step;  // (no part without values)
  if (workspace_bytes < 16L * p.batch * a.parts) {
    set_error("carekv_verify_drafts: workspace too small (%lld < %lld)", (long long)workspace_bytes,
              (long long)(16L * p.batch * a.parts));
    return CAREKV_ESPACE;
  }
  CAREKV_REQUIRE(((uintptr_t)workspace & 7) == 0, "workspace must be 8-byte aligned");
  hipStream_t s = (hipStream_t)stream;
  auto go = [&](auto e) {
    using E = decltype(e);
    hipLaunchKernelGGL(verify_sums_kernel<E>, dim3(a.parts, p.batch), dim3(256), 0, s, a);
    hipLaunchKernelGGL(verify_pick_kernel<E>, dim3(p.batch), dim3(256), 0, s, a);
  };
  if (p.dtype == CAREKV_F16) go(_Float16{});
  else if (p.dtype == CAREKV_BF16) go(__bf16{});
  else go(float{});
  CAREKV_CHECK_LAUNCH("verify_drafts");
  return CAREKV_OK;
}
