// New tokens into pages of 4-bit rows, q and k under rotary positions on the way
// (append_pages): for pair i of a head and position p, t = p f_i,
//   y1 = a (x1 cos t - x2 sin t),  y2 = a (x2 cos t + x1 sin t),
// then per 32 values s = half(max|y| / 7), c = clamp(rint(half(y / s)), -8, 7).
//
// Angles and products are 64 bits, rounded to 32 and then to the type: a product
// rounded to 32 bits first puts one k in some 10^6 into the neighbouring code,
// which is a seventh of the group's largest value.
//
// Bound by memory: each value is read and written once.  A work-group takes 4
// (D = 64: 8) consecutive places of a sequence, whose sines and cosines its
// threads compute once, one each, and its waves walk over the heads; a lane owns
// 8 dims of one token, so that the angles stay in registers over the walk.
// V's words hold four tokens of a dim: the places of a wave start at a multiple
// of four, so that no other wave writes a word of it, and a word of which only
// some tokens are new is read and joined.
//
// Measured in a graph, D = 128: 4 x 8192 tokens of 40 / 40 heads with the values
// they stand for 434 us, 5.1 TB/s, a copy's rate; of 32 / 8 heads 169, 5.0 TB/s;
// K and V alone (16 x 8192 tokens of 8 heads) 179 us at 3.9 TB/s of coding, and 223
// with positions, a token's 64-bit angles over few heads.  Divisions, and V's codes
// in bytes in LDS, took 467, 179, 222 and 268.  One token of 32 / 4 heads: 5 us.
#include <algorithm>

#include "common.h"
#include "host_util.h"
#include "pages4.h"

namespace carekv {

struct AppendArgs {
  const char* q;
  const char* k;
  const char* v;
  char* qo;
  uint16_t* k_hat;       // [B][Hkv][T][D], or null
  uint16_t* v_hat;
  const void* pos;       // or null: start + t
  const double* freqs;
  const int32_t* start;
  const int32_t* counts; // or null: T
  const int32_t* table;
  char* pages;
  long pos_batch, table_sb, q_sb, q_sh, q_st, k_sb, k_sh, k_st, v_sb, v_sh, v_st, o_sb, o_sh, o_st;  // (q .. o: bytes)
  int T, Hq, Hkv, R, nu, n_pages, max_pages, pos64, interleaved;
  int partner_wide;      // the other halves of a lane's pairs are one aligned run
  float scale;
};

// 8 elements at p: one 16-byte load where the host checked the alignment
template <typename E, bool W>
__device__ __forceinline__ void load8(E* x, const char* p, bool wide = true) {
  if (W && wide) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    __builtin_memcpy(x, &v, 16);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = reinterpret_cast<const E*>(p)[i];
  }
}

// x / s rounded to fp16, s and x fp16 values, r within 2 ulps of 1 / s: x r, and its exact rest times r.  What comes out is
// the quotient within 2^-24 (1 + 2^-20) of itself, and the quotient itself where it has at most 24 bits; other quotients
// of 11-bit numbers keep 2^-23 of themselves away from the borders of fp16's rounding, numbers of 12 bits.
__device__ __forceinline__ _Float16 half_quotient(float x, float s, float r) {
  const float q = x * r;
  return (_Float16)fmaf(fmaf(-q, s, x), r, q);
}

// A lane's 8 fp16 values as codes: p[i], codes 2i and 2i + 1 as u = c + 8 in the low bits of the halves of fp16 1024 + u;
// and the group's scale (its 4 lanes, neighbours, hold the other values).
struct Coded {
  uint32_t p[4];
  _Float16 s;
  // the codes in 4 bits each, in a word's order
  __device__ __forceinline__ uint32_t word() const {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= (p[i] & 0x000f000fu) << (4 * i);
    return w;
  }
  // what they stand for
  __device__ __forceinline__ void values(half2_t* x) const {
    const half2_t off = {(_Float16)-1032.f, (_Float16)-1032.f}, s2 = {s, s};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      half2_t h;
      __builtin_memcpy(&h, &p[i], 4);
      x[i] = (h + off) * s2;
    }
  }
};
__device__ __forceinline__ Coded code8(const _Float16* x) {
  typedef uint16_t ushort2_t __attribute__((ext_vector_type(2)));
  ushort2_t m2 = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    ushort2_t b;
    __builtin_memcpy(&b, x + 2 * i, 4);
    m2 = __builtin_elementwise_max(m2, b & (uint16_t)0x7fff);
  }
  uint32_t m = max((uint32_t)m2.x, (uint32_t)m2.y);
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xf, 0xf, false));  // lane ^ 1
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xf, 0xf, false));  // lane ^ 2
  Coded r;
  const bool bad = m >= 0x7c00;
  r.s = half_quotient(h2f((uint16_t)m), 7.f, 1.f / 7.f);
  const float s = (float)r.s, inv = s != 0.f ? __builtin_amdgcn_rcpf(s) : 0x1p60f;  // (s = 0: x 2^60, 0 or past every code)
  const half2_t lo = {(_Float16)-8.f, (_Float16)-8.f}, hi = {(_Float16)7.f, (_Float16)7.f}, up = {(_Float16)1032.f, (_Float16)1032.f};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    half2_t h = {half_quotient((float)x[2 * i], s, inv), half_quotient((float)x[2 * i + 1], s, inv)};
    h = __builtin_elementwise_min(__builtin_elementwise_max(h, lo), hi) + up;  // (rounded to whole numbers, ties to even)
    __builtin_memcpy(&r.p[i], &h, 4);
    if (bad) r.p[i] = 0x64086408u;
  }
  if (bad) r.s = bits2half(0x7e00);
  return r;
}

template <typename E, int D, bool W>
__global__ __launch_bounds__(256) void append_pages_kernel(AppendArgs a) {
  using P = Page4<D>;
  constexpr int CH = D / 8, TPW = 64 / CH;  // lanes of a token, tokens of a wave
  __shared__ double2 tab[256];              // [TPW][D / 2] cosine, sine
  __shared__ __align__(16) uint32_t codes[4][64];  // a wave's words of V's codes, as K's: [token quads][CH][4 tokens]
  const int b = blockIdx.x / a.nu, unit = blockIdx.x - b * a.nu;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int start = min(max(a.start[b], -(1 << 29)), 1 << 29);
  const int slot0 = (start & ~(TPW - 1)) + unit * TPW;
  if (slot0 >= start + a.T) return;
  const int count = min(a.counts ? a.counts[b] : a.T, a.T);
  const int half = a.R / 2;
  {
    const int i = threadIdx.x % (D / 2), t = slot0 + (int)threadIdx.x / (D / 2) - start;
    if (i < half && t >= 0 && t < a.T) {
      const long pi = b * a.pos_batch + t;
      const double p = !a.pos ? (double)((long)a.start[b] + t)
                              : a.pos64 ? (double)reinterpret_cast<const int64_t*>(a.pos)[pi]
                                        : (double)reinterpret_cast<const int32_t*>(a.pos)[pi];
      // t less its whole turns (2 pi in two parts), in half turns
      const double x = p * a.freqs[i], n = rint(x * 0.15915494309189533577);
      const double r = fma(-n, 2.4492935982947064e-16, fma(-n, 6.283185307179586477, x));
      double s, c;
      sincospi(r * 0.31830988618379067154, &s, &c);
      tab[threadIdx.x] = make_double2(c * (double)a.scale, s * (double)a.scale);
    }
  }
  __syncthreads();
  const int j = lane / CH, c = lane % CH, slot = slot0 + j, t = slot - start;
  const bool in = t >= 0 && t < a.T, fresh = t >= 0 && t < count;
  // y[e] = x[e] cs[e] + x[partner] sn[e]
  double cs[8], sn[8];
  const bool rot = 8 * c < a.R;
  // (half: a lane's dims may lie in both halves or behind R where R is no multiple of 16)
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int d = 8 * c + e;
    const int i = a.interleaved ? d / 2 : d < half ? d : d - half;
    const bool second = a.interleaved ? d & 1 : d >= half;
    const double2 w = tab[j * (D / 2) + min(i, D / 2 - 1)];
    cs[e] = d < a.R ? w.x : 1.0;
    sn[e] = d < a.R ? (second ? w.y : -w.y) : 0.0;
  }
  auto turned = [&](float* y, const E* x, const char* row) {
    E o[8];
    if (rot) {
      if (a.interleaved) {
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = x[e ^ 1];
      } else if (a.partner_wide) {
        load8<E, W>(o, row + 2 * (8 * c < half ? 8 * c + half : 8 * c - half));
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int d = 8 * c + e;
          o[e] = reinterpret_cast<const E*>(row)[d >= a.R ? d : d < half ? d + half : d - half];
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      y[e] = 8 * c + e < a.R ? (float)fma((double)(float)x[e], cs[e], (double)(float)o[e] * sn[e]) : (float)x[e];
  };
  const int page = slot0 >= 0 && slot0 / kPage < a.max_pages ? a.table[b * a.table_sb + slot0 / kPage] : -1;
  const bool there = page >= 0 && page < a.n_pages;
  for (int w = blockIdx.y * 4 + wave; w < a.Hkv + a.Hq; w += 4 * gridDim.y) {
    if (w >= a.Hkv) {
      if (!in) continue;
      const int h = w - a.Hkv;
      const char* row = a.q + b * a.q_sb + h * a.q_sh + t * a.q_st;
      E x[8], z[8];
      float y[8];
      load8<E, W>(x, row + 16 * c);
      turned(y, x, row);
#pragma unroll
      for (int e = 0; e < 8; ++e) z[e] = (E)y[e];
      char* dst = a.qo + b * a.o_sb + h * a.o_sh + t * a.o_st + 16 * c;
      if (W) {
        uint4 u;
        __builtin_memcpy(&u, z, 16);
        *reinterpret_cast<uint4*>(dst) = u;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) reinterpret_cast<E*>(dst)[e] = z[e];
      }
      continue;
    }
    char* block = a.pages + ((long)page * a.Hkv + w) * P::kBytes;
    _Float16 kx[8], vx[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) kx[e] = vx[e] = (_Float16)0.f;
    if (fresh) {
      const char* krow = a.k + b * a.k_sb + w * a.k_sh + t * a.k_st;
      const char* vrow = a.v + b * a.v_sb + w * a.v_sh + t * a.v_st;
      E x[8], z[8];
      float y[8];
      load8<E, W>(x, krow + 16 * c);
      load8<E, W>(z, vrow + 16 * c);
      turned(y, x, krow);
#pragma unroll
      for (int e = 0; e < 8; ++e) { kx[e] = (_Float16)y[e]; vx[e] = (_Float16)(float)z[e]; }
    }
    const Coded kc = code8(kx), vc = code8(vx);
    if (a.k_hat && in) {
      const long at = (((long)b * a.Hkv + w) * a.T + t) * D + 8 * c;
      half2_t h[4];
      uint4 u;
      kc.values(h);
      __builtin_memcpy(&u, h, 16);
      *reinterpret_cast<uint4*>(a.k_hat + at) = u;
      vc.values(h);
      __builtin_memcpy(&u, h, 16);
      *reinterpret_cast<uint4*>(a.v_hat + at) = u;
    }
    if (!there) continue;  // (the same for the whole wave)
    const int place = slot & (kPage - 1);
    if (fresh) {
      *reinterpret_cast<uint32_t*>(block + place * (D / 2) + 4 * c) = kc.word();
      if ((c & 3) == 0) {
        *reinterpret_cast<uint16_t*>(block + P::kKS + ((c >> 2) * kPage + place) * 2) = half2bits(kc.s);
        *reinterpret_cast<uint16_t*>(block + P::kVS + (((place >> 2) * P::G + (c >> 2)) * 4 + (place & 3)) * 2) = half2bits(vc.s);
      }
    }
    uint32_t* mine = codes[wave];
    lds_sync_wave();  // (the last head's words have been read)
    mine[((j / 4) * CH + c) * 4 + j % 4] = vc.word();
    lds_sync_wave();
    // lane: word lane % (D / 2) of token quad lane / (D / 2), dims d and d + 16 of its four tokens
    constexpr int WQ = D / 2;  // words of a quad
    const int quad = lane / WQ, l = lane % WQ, d = 32 * (l % P::G) + l / P::G;
    const int s0 = slot0 + 4 * quad - start;  // the quad's first token
    const uint4 w0 = *reinterpret_cast<const uint4*>(mine + (quad * CH + d / 8) * 4);
    const uint4 w1 = *reinterpret_cast<const uint4*>(mine + (quad * CH + d / 8 + 2) * 4);
    const uint32_t from[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
    uint32_t word = 0, put = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      word |= (from[e] >> nib4(d % 8) & 15u) << nib4(e);
      if (s0 + e % 4 >= 0 && s0 + e % 4 < count) put |= 15u << nib4(e);
    }
    if (put) {
      uint32_t* dst = reinterpret_cast<uint32_t*>(block + P::kV + (((slot0 + 4 * quad) & (kPage - 1)) / 4) * (WQ * 4)) + l;
      if (put != ~0u) word = (word & put) | (*dst & ~put);
      *dst = word;
    }
  }
}

}  // namespace carekv

using namespace carekv;

extern "C" int64_t carekv_page4_bytes(int32_t head_dim) {
  return head_dim == 64 ? Page4<64>::kBytes : head_dim == 128 ? Page4<128>::kBytes : -1;
}

extern "C" int carekv_append_pages(const carekv_append_params* pp, const void* q, const void* k, const void* v,
                                   const void* positions, const double* freqs, const int32_t* start,
                                   const int32_t* counts, const int32_t* table, void* pages, void* q_out,
                                   void* k_hat, void* v_hat, void* stream) {
  CAREKV_REQUIRE(pp, "null argument");
  const carekv_append_params& p = *pp;
  CAREKV_REQUIRE(p.head_dim == 64 || p.head_dim == 128, "head_dim must be 64 or 128");
  CAREKV_REQUIRE(p.dtype == CAREKV_F16 || p.dtype == CAREKV_BF16, "dtype must be CAREKV_F16 or CAREKV_BF16");
  CAREKV_REQUIRE(p.batch >= 0 && p.seq_len >= 0 && p.n_heads >= 0 && p.n_kv_heads > 0 && p.n_pages >= 0 && p.max_pages >= 0,
                 "negative counts");
  CAREKV_REQUIRE(p.rotary_dim >= 0 && p.rotary_dim % 2 == 0 && p.rotary_dim <= p.head_dim,
                 "rotary_dim must be even, 0 <= rotary_dim <= head_dim");
  CAREKV_REQUIRE(p.pos_bits == 32 || p.pos_bits == 64 || !positions, "pos_bits must be 32 or 64");
  CAREKV_REQUIRE(p.seq_len < (1 << 29) && p.max_pages < (1 << 25), "seq_len must be below 2^29, max_pages below 2^25");
  if (p.batch == 0 || p.seq_len == 0) return CAREKV_OK;
  CAREKV_REQUIRE(k && v && start && (p.rotary_dim == 0 || freqs) && (p.n_heads == 0 || (q && q_out)) &&
                     (p.max_pages == 0 || table) && (p.n_pages == 0 || pages) && !k_hat == !v_hat, "null argument");
  CAREKV_REQUIRE((((uintptr_t)pages | (uintptr_t)k_hat | (uintptr_t)v_hat) & 15) == 0, "pages, k_hat and v_hat must be 16-byte aligned");
  // the bytes from an operand's first value to behind its last
  auto apart = [&](const void* x, int heads, int64_t sb, int64_t sh, int64_t st) {
    const int64_t reach = 2 * ((p.batch - 1) * sb + (heads - 1) * sh + (p.seq_len - 1) * st + p.head_dim);
    const uintptr_t lo = (uintptr_t)pages, hi = lo + (uintptr_t)p.n_pages * p.n_kv_heads * carekv_page4_bytes(p.head_dim);
    return (uintptr_t)x >= hi || (uintptr_t)x + reach <= lo;
  };
  CAREKV_REQUIRE(apart(k, p.n_kv_heads, p.k_sb, p.k_sh, p.k_st) && apart(v, p.n_kv_heads, p.v_sb, p.v_sh, p.v_st) &&
                     (p.n_heads == 0 || apart(q, p.n_heads, p.q_sb, p.q_sh, p.q_st)), "k, v and q must not overlap the pages");
  AppendArgs a{};
  a.q = (const char*)q; a.k = (const char*)k; a.v = (const char*)v; a.qo = (char*)q_out;
  a.k_hat = (uint16_t*)k_hat; a.v_hat = (uint16_t*)v_hat;
  a.pos = positions; a.freqs = freqs; a.start = start; a.counts = counts; a.table = table; a.pages = (char*)pages;
  a.pos_batch = p.pos_batch; a.table_sb = p.table_sb;
  a.q_sb = 2 * p.q_sb; a.q_sh = 2 * p.q_sh; a.q_st = 2 * p.q_st; a.k_sb = 2 * p.k_sb; a.k_sh = 2 * p.k_sh; a.k_st = 2 * p.k_st;
  a.v_sb = 2 * p.v_sb; a.v_sh = 2 * p.v_sh; a.v_st = 2 * p.v_st; a.o_sb = 2 * p.qo_sb; a.o_sh = 2 * p.qo_sh; a.o_st = 2 * p.qo_st;
  const int tpw = 64 / (p.head_dim / 8);
  a.T = p.seq_len; a.Hq = p.n_heads; a.Hkv = p.n_kv_heads; a.R = p.rotary_dim; a.n_pages = p.n_pages; a.max_pages = p.max_pages;
  a.pos64 = p.pos_bits == 64; a.interleaved = p.interleaved != 0; a.scale = p.scale;
  a.nu = (p.seq_len + 2 * tpw - 2) / tpw;
  uintptr_t bits = operand_bits(k, {{p.batch, a.k_sb}, {p.n_kv_heads, a.k_sh}, {p.seq_len, a.k_st}}) |
                   operand_bits(v, {{p.batch, a.v_sb}, {p.n_kv_heads, a.v_sh}, {p.seq_len, a.v_st}});
  if (p.n_heads)
    bits |= operand_bits(q, {{p.batch, a.q_sb}, {p.n_heads, a.q_sh}, {p.seq_len, a.q_st}}) |
            operand_bits(q_out, {{p.batch, a.o_sb}, {p.n_heads, a.o_sh}, {p.seq_len, a.o_st}});
  const bool wide = (bits & 15) == 0;
  a.partner_wide = wide && p.rotary_dim % 16 == 0;
  const long units = (long)p.batch * a.nu;
  CAREKV_REQUIRE(grid_fits(units, 256), "too many tokens");
  const long heads = (long)p.n_heads + p.n_kv_heads;
  CAREKV_REQUIRE(heads < 65536, "too many heads");
  // walks cut until 1024 work-groups (4 a CU) are there
  const long cuts = std::max(1L, std::min((heads + 3) / 4, 1024 / units));
  const dim3 grid((unsigned)units, (unsigned)cuts);
  hipStream_t s = (hipStream_t)stream;
  const int rc = dispatch_elem_d(p.dtype, p.head_dim, [&](auto et, auto d) {
    using E = typename decltype(et)::E;
    constexpr int D = decltype(d)::value;
    if (wide) hipLaunchKernelGGL((append_pages_kernel<E, D, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((append_pages_kernel<E, D, false>), grid, dim3(256), 0, s, a);
    return CAREKV_OK;
  });
  CAREKV_CHECK_LAUNCH("append_pages");
  return rc;
}
