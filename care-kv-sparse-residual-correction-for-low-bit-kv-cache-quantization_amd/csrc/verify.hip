// Drafted tokens against the model's probabilities (verify_drafts): token x_t of
// a sequence is accepted while u_t q_t(x_t) < p_t(x_t), and behind the n accepted
// ones comes the smallest i with
//   w_0 + .. + w_i > u_next (w_0 + .. + w_(V-1)),
// w = max(p_n - q_n, 0) where a token was rejected (and any w is over 0), else
// p_n.  Products and sums are 64 bits: the order of their rounding moves a border
// between tokens by 2^-50 of the sum, in 32 bits by as much as a token holds.
//
// Bound by reading the one row of p and q that the next token is drawn from.  A
// row is cut into segments of 1024 values, whose sums a wave takes each (sixteen
// values a lane, all in flight); from the segments' sums one wave finds the
// segment and then the place in it.  Two launches, the first over the whole GPU;
// short rows do both in one work-group a sequence, which saves a launch.
// Measured in a graph (fp32, both p and q, 8 drafts): 128 x 131071, 134 MB in
// 30.3 us (4.4 TB/s; one work-group a sequence 32.0), 1 x 131071 11.7 (25.9),
// 16 x 65536 10.7 (16.1), 16 x 16384 10.4 (9.5), 1 x 2048 8.9 (7.0).  What is
// left of a short row is the chain of dependent loads: the draft, its
// probabilities, the row, the segment.
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
  double2* sums;         // [B][segs]: of max(p - q, 0), of p; null with one launch
  long p_sb, p_st, q_sb, q_st, draft_sb, u_sb;  // elements
  int T, V, segs;
};

constexpr int kSeg = 1024;      // values of a segment
constexpr int kSegsInLds = 32; // at most: two for each wave of a work-group

// How many of sequence b's tokens are accepted (every wave for itself).
template <typename E>
__device__ __forceinline__ int count_accepted(const VerifyArgs& a, int b, int count) {
  int n = 0;
  for (; n < count; n += 64) {
    const int t = n + (threadIdx.x & 63);
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
  return min(n, count);
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
  __device__ __forceinline__ void of(int i, double v, double less, double& r, double& w) const {
    const double d = i == x ? 0.0 : v - less;
    w = v > 0.0 ? v : 0.0;
    r = rest ? (d > 0.0 ? d : 0.0) : w;
  }
  __device__ __forceinline__ void at(int i, double& r, double& w) const {
    of(i, (double)(float)p[i], q ? (double)(float)q[i] : 0.0, r, w);
  }
};

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// The sums of segment seg, by a wave: sixteen loads of each row in flight.
template <typename E>
__device__ __forceinline__ double2 segment_sums(const VerifyArgs& a, const Weights<E>& w, int seg) {
  const int lane = threadIdx.x & 63, i0 = seg * kSeg + lane;
  double r = 0.0, s = 0.0;
  if (i0 - lane + kSeg <= a.V) {
    E p[kSeg / 64], q[kSeg / 64];
#pragma unroll
    for (int k = 0; k < kSeg / 64; ++k) p[k] = w.p[i0 + 64 * k];
    if (w.q)
#pragma unroll
      for (int k = 0; k < kSeg / 64; ++k) q[k] = w.q[i0 + 64 * k];
#pragma unroll
    for (int k = 0; k < kSeg / 64; ++k) {
      double x, y;
      w.of(i0 + 64 * k, (double)(float)p[k], w.q ? (double)(float)q[k] : 0.0, x, y);
      r += x;
      s += y;
    }
  } else {
    for (int i = i0; i < a.V; i += 64) {
      double x, y;
      w.at(i, x, y);
      r += x;
      s += y;
    }
  }
  return make_double2(wave_sum_d(r), wave_sum_d(s));
}

// The first of the wave's 64 runs (lane by lane) at whose end the sum passes the goal, of those with any weight; where
// none does (a number of 1 and more), the last one.  base: the sum before it.  -1: no run has any.
__device__ __forceinline__ int find_run(double mine, double before, double goal, double& base) {
  double end = mine;  // inclusive
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double x = __shfl_up(end, o, 64);
    if ((int)(threadIdx.x & 63) >= o) end += x;
  }
  const unsigned long long some = __ballot(mine > 0.0), past = __ballot(mine > 0.0 && before + end > goal);
  const int who = past ? __ffsll((long long)past) - 1 : some ? 63 - __clzll((long long)some) : -1;
  base = before + __shfl(end - mine, max(who, 0), 64);
  return who;
}

// The token behind the accepted ones, by a wave, from the segments' sums.
template <typename E>
__device__ __forceinline__ int pick_token(const VerifyArgs& a, const Weights<E>& w, const double2* sums, float u) {
  const int lane = threadIdx.x & 63, per = (a.segs + 63) / 64, s0 = min(lane * per, a.segs), s1 = min(s0 + per, a.segs);
  double r = 0.0, s = 0.0;
  for (int i = s0; i < s1; ++i) {
    const double2 x = sums[i];
    r += x.x;
    s += x.y;
  }
  const double all_r = wave_sum_d(r), all_s = wave_sum_d(s);
  const bool rest = all_r > 0.0;
  double goal = (double)u * (rest ? all_r : all_s), base;
  if (!(goal >= 0.0)) goal = 0.0;
  const int who = find_run(rest ? r : s, 0.0, goal, base);
  if (who < 0) return -1;
  // the segment among that lane's
  int seg = -1;
  double at = base, before = base;
  for (int i = s0; i < s1; ++i) {
    const double x = rest ? sums[i].x : sums[i].y;
    if (x > 0.0) {
      seg = i;
      before = at;
      if (at + x > goal) break;
    }
    at += x;
  }
  seg = __shfl(seg, who, 64);
  before = __shfl(before, who, 64);
  // sixteen values a lane, and the place among those of the lane that passes the goal
  const int i0 = seg * kSeg + lane * (kSeg / 64);
  double v[kSeg / 64], mine = 0.0;
#pragma unroll
  for (int k = 0; k < kSeg / 64; ++k) {
    double x = 0.0, y = 0.0;
    if (i0 + k < a.V) w.at(i0 + k, x, y);
    v[k] = rest ? x : y;
    mine += v[k];
  }
  const int lane_of = find_run(mine, before, goal, base);
  int token = -1;
  bool done = false;
  at = base;
#pragma unroll
  for (int k = 0; k < kSeg / 64; ++k) {
    at += v[k];
    if (v[k] > 0.0 && !done) {
      token = i0 + k;
      done = at > goal;
    }
  }
  return __shfl(token, max(lane_of, 0), 64);
}

// Sequence b's results, by a wave.
__device__ __forceinline__ void write_verdict(const VerifyArgs& a, int b, int n, int token) {
  for (int t = threadIdx.x & 63; t <= a.T; t += 64)
    a.tokens[(long)b * (a.T + 1) + t] = t < n ? (int32_t)a.draft[b * a.draft_sb + t] : t == n ? token : -1;
  if ((threadIdx.x & 63) == 0) a.accepted[b] = n;
}

__device__ __forceinline__ int count_of(const VerifyArgs& a, int b) {
  return a.counts ? min(max(a.counts[b], 0), a.T) : a.T;
}

template <typename E>
__global__ __launch_bounds__(256) void verify_sums_kernel(VerifyArgs a) {
  const int b = blockIdx.y, count = count_of(a, b), n = count_accepted<E>(a, b, count);
  const Weights<E> w(a, b, n, count);
  for (int seg = blockIdx.x * 4 + (threadIdx.x >> 6); seg < a.segs; seg += 4 * gridDim.x) {
    const double2 x = segment_sums(a, w, seg);
    if ((threadIdx.x & 63) == 0) a.sums[(long)b * a.segs + seg] = x;
  }
}

template <typename E>
__global__ __launch_bounds__(64) void verify_pick_kernel(VerifyArgs a) {
  const int b = blockIdx.x, count = count_of(a, b), n = count_accepted<E>(a, b, count);
  const Weights<E> w(a, b, n, count);
  write_verdict(a, b, n, pick_token(a, w, a.sums + (long)b * a.segs, a.u_next[b]));
}

template <typename E>
__global__ __launch_bounds__(1024) void verify_kernel(VerifyArgs a) {
  __shared__ double2 s_sums[kSegsInLds];
  const int b = blockIdx.x, count = count_of(a, b), n = count_accepted<E>(a, b, count);
  const Weights<E> w(a, b, n, count);
  for (int seg = threadIdx.x >> 6; seg < a.segs; seg += 16) {
    const double2 x = segment_sums(a, w, seg);
    if ((threadIdx.x & 63) == 0) s_sums[seg] = x;
  }
  __syncthreads();
  if (threadIdx.x < 64) write_verdict(a, b, n, pick_token(a, w, s_sums, a.u_next[b]));
}

namespace {
int verify_segs(const carekv_verify_params& p) { return (p.vocab + kSeg - 1) / kSeg; }
// One work-group a sequence where each of its waves has at most two segments and each CU at most one work-group; else two
// launches.  In a graph (us, one launch against two): 128 x 16384 9.7 to 11.2, 1 x 32000 11.3 to 10.0, 1 x 65536 14.9 to
// 9.3, 512 x 4096 15.1 to 11.2.  Called eagerly, the second launch and its workspace cost the host another 4 us (1 x 32000:
// 11.5 to 15.8), so the border is where one launch loses less than that.
bool verify_fused(const carekv_verify_params& p) { return verify_segs(p) <= kSegsInLds && p.batch <= 256; }
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
  return verify_fused(*pp) ? 0 : 16L * pp->batch * verify_segs(*pp);
}

extern "C" int carekv_verify_drafts(const carekv_verify_params* pp, const int64_t* draft, const void* target_probs,
                                    const void* draft_probs, const float* u, const float* u_next,
                                    const int32_t* counts, int32_t* tokens, int32_t* accepted, void* workspace,
                                    int64_t workspace_bytes, void* stream) {
  const int rc = check_verify(pp);
  if (rc != CAREKV_OK) return rc;
  const carekv_verify_params& p = *pp;
  if (p.batch == 0) return CAREKV_OK;
  CAREKV_REQUIRE(target_probs && u_next && tokens && accepted && (workspace || verify_fused(p)) && (p.n_drafts == 0 || (draft && u)), "null argument");
  VerifyArgs a{};
  a.p = (const char*)target_probs; a.q = p.n_drafts ? (const char*)draft_probs : nullptr; a.draft = draft; a.u = u;
  a.u_next = u_next; a.counts = counts; a.tokens = tokens; a.accepted = accepted; a.sums = (double2*)workspace;
  a.p_sb = p.target_sb; a.p_st = p.target_st; a.q_sb = p.draft_probs_sb; a.q_st = p.draft_probs_st;
  a.draft_sb = p.draft_sb; a.u_sb = p.u_sb;
  a.T = p.n_drafts; a.V = p.vocab; a.segs = verify_segs(p);
  const bool fused = verify_fused(p);
  const int64_t need = carekv_verify_drafts_workspace_bytes(pp);
  if (workspace_bytes < need) {
    set_error("carekv_verify_drafts: workspace too small (%lld < %lld)", (long long)workspace_bytes, (long long)need);
    return CAREKV_ESPACE;
  }
  CAREKV_REQUIRE(((uintptr_t)workspace & 15) == 0, "workspace must be 16-byte aligned");
  hipStream_t s = (hipStream_t)stream;
  // work-groups of a sequence: each wave a segment, until 2048 of them are there (256 x 131071: 41.1 us, with 1024 43.7,
  // with 4096 40.8)
  const int wgs = std::max(1, std::min((a.segs + 3) / 4, 2048 / p.batch));
  auto go = [&](auto e) {
    using E = decltype(e);
    if (fused) {
      hipLaunchKernelGGL(verify_kernel<E>, dim3(p.batch), dim3(1024), 0, s, a);
      return;
    }
    hipLaunchKernelGGL(verify_sums_kernel<E>, dim3(wgs, p.batch), dim3(256), 0, s, a);
    hipLaunchKernelGGL(verify_pick_kernel<E>, dim3(p.batch), dim3(64), 0, s, a);
  };
  if (p.dtype == CAREKV_F16) go(_Float16{});
  else if (p.dtype == CAREKV_BF16) go(__bf16{});
  else go(float{});
  CAREKV_CHECK_LAUNCH("verify_drafts");
  return CAREKV_OK;
}
