// Shared pieces of the gated projection (gated.hip): element types, the activation, the saved pre-activations.
#pragma once
#include "common.h"

namespace cagc {
namespace gated {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
struct e4m3 { uint8_t v; };

template <class T> struct Type;      // bytes of an element
template <> struct Type<float> { static constexpr int size = 4; };
template <> struct Type<_Float16> { static constexpr int size = 2; };
template <> struct Type<__bf16> { static constexpr int size = 2; };
template <> struct Type<e4m3> { static constexpr int size = 1; };

// One matrix-core step over the 128 bytes of K that a stage holds of a row.  A lane brings the 16-byte chunks number lane/16 and
// 4 + lane/16 of its row (lane % 16) of either operand; which k a chunk's elements are does not matter as long as both operands
// agree, so one addressing serves 2 products of 16x16x32 (16-bit), 8 of 16x16x4 (fp32) and 1 of 16x16x128 (e4m3).
template <class T> __device__ __forceinline__ f32x4 mma(const i32x4 (&a)[2], const i32x4 (&b)[2], f32x4 c);
template <> __device__ __forceinline__ f32x4 mma<__bf16>(const i32x4 (&a)[2], const i32x4 (&b)[2], f32x4 c) {
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a[0]), __builtin_bit_cast(bf16x8, b[0]), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a[1]), __builtin_bit_cast(bf16x8, b[1]), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x4 mma<_Float16>(const i32x4 (&a)[2], const i32x4 (&b)[2], f32x4 c) {
  c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a[0]), __builtin_bit_cast(f16x8, b[0]), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a[1]), __builtin_bit_cast(f16x8, b[1]), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x4 mma<float>(const i32x4 (&a)[2], const i32x4 (&b)[2], f32x4 c) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const f32x4 x = __builtin_bit_cast(f32x4, a[h]), y = __builtin_bit_cast(f32x4, b[h]);
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], c, 0, 0, 0);
  }
  return c;
}
template <> __device__ __forceinline__ f32x4 mma<e4m3>(const i32x4 (&a)[2], const i32x4 (&b)[2], f32x4 c) {
  const i32x8 x = __builtin_shufflevector(a[0], a[1], 0, 1, 2, 3, 4, 5, 6, 7), y = __builtin_shufflevector(b[0], b[1], 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 0, 0, 0, 0, 0, 0);      // both e4m3, no block scales
}

// act(g) and act'(g).  SiLU: g s with s = 1 / (1 + e^-g), derivative s (1 + g (1 - s)); GELU: g Phi(g), derivative Phi(g) + g phi(g).
__device__ __forceinline__ float act_of(int act, float g) {
  if (act == CAGC_ACT_SILU) return g * __builtin_amdgcn_rcpf(1.f + __expf(-g));
  return 0.5f * g * (1.f + erff(g * 0.70710678118654752f));
}
__device__ __forceinline__ void act_grad(int act, float g, float& a, float& da) {
  if (act == CAGC_ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.f + __expf(-g));
    a = g * s;
    da = s * (1.f + g * (1.f - s));
    return;
  }
  const float c = 0.5f * (1.f + erff(g * 0.70710678118654752f));
  a = g * c;
  da = c + g * __expf(-0.5f * g * g) * 0.39894228040143268f;
}

// Saved pre-activations.  fp32: two planes [rows, n].  16-bit types: the upper 24 bits of each fp32 value, as three 16-bit planes (the
// upper halves of g, of u, and the two third bytes).  Rounding them to the input's type instead (2 planes) would add an error as
// large as that of the gradients' own rounding: measured against 64 bits, the gradients' error in bf16 is 1.4 times that of one
// final rounding with 24 bits and 1.8 times with 16.
__device__ __forceinline__ uint32_t top24(float v) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v);
  return (b & 0x7fffffffu) > 0x7f800000u ? 0x7fc000u : (b + 0x80u) >> 8;
}
__device__ __forceinline__ float from24(uint32_t hi, uint32_t lo) { return __builtin_bit_cast(float, (hi << 16) | (lo << 8)); }

}  // namespace gated
}  // namespace cagc
