// Division by a number that the host knows, in kernels whose first loads wait
// for their work-group's place: the GPU has no integer division, a 32-bit one
// is some 30 dependent instructions and a 64-bit one over 100.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace carekv {

// x / d for 0 <= x < 2^31 and 0 < d < 2^31: with 2^l the power of two not below
// d and m = floor(2^32 (2^l - d) / d) + 1, x / d = (hi32(m x) + x) >> l (Granlund
// and Montgomery, Division by Invariant Integers using Multiplication, 1994; their
// sum passes 32 bits only for larger x).
struct FastDiv {
  uint32_t m, l;
  int d;
  FastDiv() = default;
  explicit FastDiv(int64_t div) : d((int)div) {
    l = 0;
    while ((1ull << l) < (uint64_t)div) ++l;
    m = (uint32_t)(((1ull << 32) * ((1ull << l) - (uint64_t)div)) / (uint64_t)div + 1);
  }
};
__host__ __device__ __forceinline__ int operator/(int x, const FastDiv& f) {
  return (int)(((uint32_t)(((uint64_t)f.m * (uint32_t)x) >> 32) + (uint32_t)x) >> f.l);
}
__host__ __device__ __forceinline__ int operator%(int x, const FastDiv& f) { return x - x / f * f.d; }

// Where part i of n things starts, cut into f.d parts whose sizes differ by at most one.
__host__ __device__ __forceinline__ int part_start(int n, int i, const FastDiv& f) {
  const int q = n / f, r = n - q * f.d;
  return i * q + (i < r ? i : r);
}

}  // namespace carekv
