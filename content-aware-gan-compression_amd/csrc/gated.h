// Shared pieces of the gated projection (gated.hip): element types, the activation, the saved pre-activations.
#pragma once
#include "rows.h"

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

// One matrix-core step over the 64 bytes of K (e4m3: 128) that a piece of a stage holds of a row.  A lane brings the 16-byte chunk number lane / 16 (e4m3: and 4 + lane / 16) of
// its row (lane % 16) of either operand; which k a chunk's elements are does not matter as long as both operands agree, so one addressing serves one product of 16x16x32 (16-bit), 4 of
// 16x16x4 (fp32) and one of 16x16x128 (e4m3, no block scales).
// The accumulators are fp32.  Before it adds to them, the e4m3 instruction (the one of half its width, too) cuts each of 8 neighbouring products to a multiple of 2^-14 of the largest one's power of
// two; the 16-bit ones keep 24 bits.  Against 64 bits, rows and weights of normal values: 1.5e-5 of the sums' size at any K, where fp32 would leave 5e-8 to 1e-7; the operands' own rounding to e4m3 is 2^-4
// a value and the output's 2^-9 (bf16), so twice the time for the products on 16-bit operands is not spent on it.
template <class T> struct Piece { typedef i32x4 type; static constexpr int count = 2; };      // a lane's part of a piece; pieces in 128 bytes
template <> struct Piece<e4m3> { typedef i32x8 type; static constexpr int count = 1; };
template <class T> __device__ __forceinline__ f32x4 mma(typename Piece<T>::type a, typename Piece<T>::type b, f32x4 c);
template <> __device__ __forceinline__ f32x4 mma<__bf16>(i32x4 a, i32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x4 mma<_Float16>(i32x4 a, i32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x4 mma<float>(i32x4 a, i32x4 b, f32x4 c) {
  const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
  for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], c, 0, 0, 0);
  return c;
}
template <> __device__ __forceinline__ f32x4 mma<e4m3>(i32x8 a, i32x8 b, f32x4 c) { return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0); }
__device__ __forceinline__ i32x8 join(i32x4 a, i32x4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }

// act(g) and act'(g).  SiLU: g s with s = 1 / (1 + e^-g), derivative s (1 + g (1 - s)); GELU: g Phi(g), derivative Phi(g) + g phi(g).
// The exponential and the reciprocal are the hardware's (a step of the last place each, and the exponent's rounding: an error of s of |g| 2^-24, no more than rounding g to fp32 makes).  Against 64 bits
// SiLU's rms error is within 1.3 times that of 1 / (1 + expf(-g)) above g = -1, 1.6 down to -3, 3 to 6 below, where the values fade.
// Phi in two pieces, both computed, without branches: within 1.25 of zero 1/2 + g C(g^2), elsewhere Phi(-|g|) = e^(-g^2/2) t R(t) with t = 1 / (1 + |g| / 4), whose exponential is phi's too.  C and R are
// least-maximum fits to the two functions in 64 bits (2e-9 of Phi, 8e-9 of Phi(-|g|)); in fp32 Phi is off by at most 1.0 2^-24, and below -1.25 by about (7 + g^2) 2^-24 of itself.
__device__ __forceinline__ float normal_cdf(float g, float& e) {
  const float u = g * g, x = fabsf(g), t = __builtin_amdgcn_rcpf(1.f + 0.25f * x);
  e = __expf(-0.5f * u);
  const float c = ((((-6.645250323344953e-06f * u + 0.00011032923066522926f) * u - 0.0011827126145362854f) * u + 0.009971503168344498f) * u - 0.06648998707532883f) * u + 0.3989422619342804f;
  const float r = ((((((-0.04816504567861557f * t + 0.11408009380102158f) * t - 0.029239512979984283f) * t + 0.09755606204271317f) * t + 0.07119438052177429f) * t + 0.09522004425525665f) * t
                   + 0.09956982731819153f) * t + 0.0997423306107521f;
  const float tail = t * r * e;
  return x < 1.25f ? 0.5f + g * c : (g < 0.f ? tail : 1.f - tail);
}
__device__ __forceinline__ float act_of(int act, float g) {
  if (act == CAGC_ACT_SILU) return g * __builtin_amdgcn_rcpf(1.f + __expf(-g));
  float e;
  return g * normal_cdf(g, e);
}
__device__ __forceinline__ void act_grad(int act, float g, float& a, float& da) {
  if (act == CAGC_ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.f + __expf(-g));
    a = g * s;
    da = s * (1.f + g * (1.f - s));
    return;
  }
  float e;
  const float c = normal_cdf(g, e);
  a = g * c;
  da = c + g * e * 0.39894228040143268f;
}

// Saved pre-activations.  fp32: two planes [rows, n].  16-bit types: the upper 24 bits of each fp32 value (a significand of 16 bits, cut: within 2^-15 of the value, and a
// NaN's quiet bit stays), as three 16-bit planes: the upper halves of g, of u, and their third bytes (g's in the upper byte).  Rounding them to the input's
// type instead (2 planes) would add an error as large as that of the gradients' own rounding: against 64 bits, the gradients' error in bf16 is 1.4 times
// that of one final rounding with 24 bits and 1.8 times with 16.
__device__ __forceinline__ float from24(uint32_t hi, uint32_t lo) { return __builtin_bit_cast(float, (hi << 16) | (lo << 8)); }
__device__ __forceinline__ uint32_t bits(float v) { return __builtin_bit_cast(uint32_t, v); }
// the upper halves of two values; the third bytes of two values each of g and u
__device__ __forceinline__ uint32_t upper2(float a, float b) { return __builtin_amdgcn_perm(bits(b), bits(a), 0x07060302u); }
__device__ __forceinline__ uint32_t third2(float g0, float u0, float g1, float u1) {
  const uint32_t x = __builtin_amdgcn_perm(bits(g0), bits(u0), 0x0c0c0501u), y = __builtin_amdgcn_perm(bits(g1), bits(u1), 0x0c0c0501u);
  return x | y << 16;
}

}  // namespace gated
}  // namespace cagc
