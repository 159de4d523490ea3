// 16-bit element types of the prompt operators and their matrix products.
#pragma once

#include "decode_page.h"
#include "host_util.h"

namespace carekv {

typedef __bf16 bhalf8_t __attribute__((ext_vector_type(8)));

// kUp: a weight of 2^kUp at most is held where the largest is the row's, so that small ones stay normal (fp16: those
// down to 2^-29 of it).
struct ElemF16 {
  using E = _Float16;
  using V8 = half8_t;
  static constexpr float kUp = 15.f;
  static __device__ __forceinline__ float4_t mfma(V8 a, V8 b, float4_t c) { return mfma16x32(a, b, c); }
};
struct ElemBF16 {
  using E = __bf16;
  using V8 = bhalf8_t;
  static constexpr float kUp = 0.f;
  static __device__ __forceinline__ float4_t mfma(V8 a, V8 b, float4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994531f;
constexpr float kLowest = -3.0e38f;  // a running maximum's start: below any finite score, its own weights finite

// f(element type, std::integral_constant<int, D>) for dtype CAREKV_F16 / CAREKV_BF16 and head_dim 64 / 128
template <typename F>
int dispatch_elem_d(int dtype, int D, F&& f) {
  using I64 = std::integral_constant<int, 64>;
  using I128 = std::integral_constant<int, 128>;
  if (dtype == CAREKV_F16) return D == 64 ? f(ElemF16{}, I64{}) : f(ElemF16{}, I128{});
  return D == 64 ? f(ElemBF16{}, I64{}) : f(ElemBF16{}, I128{});
}

}  // namespace carekv
