// Pages of 4-bit rows: 16 tokens of one kv head in one block of bytes, laid out
// as the matrix instructions read them.
//
// A group of 32 values x of a row (fp16) is kept as s = half(max|x| / 7) and c =
// clamp(rint(half(x / s)), -8, 7), 0 where s and x are 0, and stands for half(c
// s); a group with a value that is not finite in fp16 stands for NaN (s = NaN, c
// = 0).  A code is held as u = c + 8 in 4 bits; of eight codes e = 0..7 in a
// 32-bit word the even ones take nibbles 0..3, the odd ones nibbles 4..7, so
// that masking one nibble out of each half of the word gives two neighbours.
//
//   K codes   [16 tokens][D / 8 words]: word w of a token's row, dims 8w + e
//   V codes   [4 token quads][16 c][D / 32 words]: word w, dims 16 (2w + e / 4) +
//             c, token e % 4 of the quad
//   V scales  [4 token quads][D / 32 groups][4 tokens] fp16
//   K scales  [D / 32 groups][16 tokens] fp16
//
// Lane 16 g + c of a wave then finds token c's dims g D / 4 .. of K in D / 8
// consecutive bytes, those of one group, and of V token quad g of the dims 16 i
// + c in as many: operands of v_mfma_f32_16x16x32 for S^T = K Q^T and O^T = V^T
// P^T without a shuffle, a wave's load being 1 KB in one piece.
#pragma once

#include "mfma16.h"

namespace carekv {

template <int D>
struct Page4 {
  static constexpr int G = D / kGroup;            // groups of a row
  static constexpr int kK = kPage * D / 2;        // bytes of K's codes
  static constexpr int kV = kK;                   // where V's codes start
  static constexpr int kVS = 2 * kK;              // V's scales
  static constexpr int kKS = kVS + kPage * G * 2; // K's scales
  static constexpr int kBytes = kKS + kPage * G * 2;
};

// Place of code e in its word, in bits.
__host__ __device__ constexpr int nib4(int e) { return 4 * ((e & 1) * 4 + (e >> 1)); }

// The codes of a word as fp16: 1024 + u in the mantissa of each half, then - 1032
// (a nibble four bits up: 1024 + 16 u, times 1 / 16, - 72), both exact; times
// their scales, rounded once as the definition has it.  s[i]: codes 2i and 2i + 1.
// The masks sit in vector registers, the exponents in a scalar one: an instruction
// takes one scalar operand and no literal, and the compiler else spends an AND and
// an OR on each pair.
struct Unpack4 {
  uint32_t lo = 0x000f000fu, hi = 0x00f000f0u, one = 0x64006400u;
  __device__ __forceinline__ Unpack4() { asm volatile("" : "+v"(lo), "+v"(hi), "+s"(one)); }
  __device__ __forceinline__ void operator()(half2_t* v, uint32_t w, const half2_t* s) const {
    const half2_t one16 = {(_Float16)0.0625f, (_Float16)0.0625f}, off = {(_Float16)-1032.f, (_Float16)-1032.f},
                  off16 = {(_Float16)-72.f, (_Float16)-72.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t bits = ((i < 2 ? w : w >> 8) & (i & 1 ? hi : lo)) | one;
      half2_t h;
      __builtin_memcpy(&h, &bits, 4);
      h = i & 1 ? __builtin_elementwise_fma(h, one16, off16) : h + off;
      v[i] = h * s[i];
    }
  }
};

}  // namespace carekv
