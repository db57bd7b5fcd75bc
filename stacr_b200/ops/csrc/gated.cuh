// The activations of gated feed-forward blocks and their derivatives in fp32, and conversions from and to the tensor types.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace sb {

enum : int { DT_BF16 = 0, DT_FP16 = 1, DT_FP32 = 2 };
enum : int { ACT_SILU = 0, ACT_GELU = 1, ACT_GELU_TANH = 2 };

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// e^x as 2^t (1 + r ln 2) with t = fl(x log2 e) and r the rounding error of that product, which one fma recovers: the library
// is compiled for fast math, whose exponential drops r and is off by |x| 2^-24.  Infinite t is left alone (r would be NaN).
__device__ __forceinline__ float exp_f32(float x) {
  const float l2e = 1.44269504f, ln2 = 0.693147181f, l2e_lo = 1.92596303e-8f;
  const float t = x * l2e;
  const float e = exp2f(t);
  const float r = fmaf(x, l2e_lo, fmaf(x, l2e, -t));
  return fabsf(t) < 126.f ? fmaf(e * ln2, r, e) : e;
}

// 1 / (1 + e^-x).  e^-x overflows to infinity below x = -88, where the result is 0.
__device__ __forceinline__ float sigmoid_f32(float x) { return __frcp_rn(1.f + exp_f32(-x)); }

// tanh z = 1 - 2 / (1 + e^2z); |z| below 2^-3 would cancel, so the odd series z - z^3/3 + 2 z^5/15 - 17 z^7/315 (next term
// 62 z^9/2835 < 2^-29 z) is used there.
__device__ __forceinline__ float tanh_f32(float z) {
  const float z2 = z * z;
  const float series = z * fmaf(z2, fmaf(z2, fmaf(z2, -0.053968254f, 0.133333333f), -0.333333333f), 1.f);
  return fabsf(z) < 0.125f ? series : 1.f - 2.f * __frcp_rn(1.f + exp_f32(2.f * z));
}

// act(x) and act'(x):
//   silu       x s,                        s (1 + x (1 - s)),      s = sigmoid(x)
//   gelu       x Phi(x),                   Phi(x) + x phi(x)       (normal distribution function and density)
//   gelu_tanh  x (1 + t) / 2,              (1 + t) / 2 + x (1 - t^2) w' / 2,   t = tanh w, w = sqrt(2/pi) (x + 0.044715 x^3)
template <int ACT>
__device__ __forceinline__ void act_and_derivative(float x, float& act, float& der) {
  if (ACT == ACT_SILU) {
    const float s = sigmoid_f32(x);
    act = x * s;
    der = s * fmaf(x, 1.f - s, 1.f);
  } else if (ACT == ACT_GELU) {
    const float cdf = 0.5f * erfcf(-0.707106781f * x);
    const float pdf = 0.398942280f * exp_f32(-0.5f * x * x);
    act = x * cdf;
    der = fmaf(x, pdf, cdf);
  } else {
    const float k = 0.797884561f, c = 0.044715f;
    const float t = tanh_f32(k * x * fmaf(c * x, x, 1.f));
    act = 0.5f * x * (1.f + t);
    der = 0.5f * (1.f + t) + 0.5f * x * (1.f - t) * (1.f + t) * k * fmaf(3.f * c * x, x, 1.f);
  }
}

// Upper 24 bits of a float, rounded; NaN and infinity keep theirs.
__device__ __forceinline__ unsigned upper24(float v) {
  const unsigned b = __float_as_uint(v);
  return (b & 0x7fffffffu) < 0x7f800000u ? b + 0x80u : b;
}

template <int ACT>
__device__ __forceinline__ float activation(float x) {
  float act, der;
  act_and_derivative<ACT>(x, act, der);
  return act;
}

}  // namespace sb
