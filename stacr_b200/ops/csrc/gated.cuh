// The activations of gated feed-forward blocks and their derivatives in fp32, and conversions from and to the tensor types.
#pragma once
#include <cuda_fp16.h>

#include <type_traits>

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

// Launches that may begin while the kernel before them in the stream drains: the launch itself and what a kernel does before
// after_predecessors() (barriers, tensor memory) are then hidden.  A launch made this way starts when every block of its
// predecessor has ended, but nothing else orders it behind that kernel's stores: so every thread calls after_predecessors(), which
// waits for the predecessor's completion, before its first access to global memory.  33 tokens of K 1536, F 8960, one call after
// another: 16.3 us without, 13.4 with; one token of K 2048, F 8192: 13.7 and 11.9.
__device__ __forceinline__ void after_predecessors() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... Params, typename... Args>
static int launch_early(void (*kernel)(Params...), dim3 grid, dim3 block, size_t shared, cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = shared;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...));
}

// VEC neighbouring values as one access, and to and from fp32 (16-bit types two at a time).
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};
template <typename T, int VEC>
__device__ __forceinline__ void unpack(const Pack<T, VEC>& p, float (&f)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) f[i] = to_f32(p.v[i]);
}
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> pack(const float (&f)[VEC]) {
  Pack<T, VEC> p;
  if constexpr (sizeof(T) == 2 && VEC > 1) {
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {
      if constexpr (std::is_same<T, __half>::value) reinterpret_cast<__half2*>(p.v)[i / 2] = __floats2half2_rn(f[i], f[i + 1]);
      else reinterpret_cast<__nv_bfloat162*>(p.v)[i / 2] = __floats2bfloat162_rn(f[i], f[i + 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) p.v[i] = from_f32<T>(f[i]);
  }
  return p;
}

// Inputs and results of the kernels never overlap, so loads may pass stores: the non-coherent path says so to the compiler.
template <typename P>
__device__ __forceinline__ P load_once(const void* p) {
  P v;
  if constexpr (sizeof(P) == 16) *reinterpret_cast<uint4*>(&v) = __ldg(static_cast<const uint4*>(p));
  else if constexpr (sizeof(P) == 8) *reinterpret_cast<uint2*>(&v) = __ldg(static_cast<const uint2*>(p));
  else if constexpr (sizeof(P) == 4) *reinterpret_cast<unsigned*>(&v) = __ldg(static_cast<const unsigned*>(p));
  else *reinterpret_cast<unsigned short*>(&v) = __ldg(static_cast<const unsigned short*>(p));
  return v;
}

// e^x as 2^t (1 + r ln 2) with t = fl(x log2 e) and r the rounding error of that product, which one fma recovers: the library
// is compiled for fast math, whose exponential drops r and is off by |x| 2^-24.  Infinite t is left alone (r would be NaN).
__device__ __forceinline__ float exp_f32(float x) {
  const float l2e = 1.44269504f, ln2 = 0.693147181f, l2e_lo = 1.92596303e-8f;
  const float t = x * l2e;
  const float e = exp2f(t);
  const float r = fmaf(x, l2e_lo, fmaf(x, l2e, -t));
  return fabsf(t) < 126.f ? fmaf(e * ln2, r, e) : e;
}

// 1 / (1 + e^-x).  e^-x overflows to infinity below x = -88, where the result is 0.  FAST: the hardware's exponential and reciprocal,
// off by (3 + 1.2 |x|) 2^-23 of the result: for results that are rounded to 16-bit types (fp16: 2^-11) or kept in 24 bits (2^-16).
__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <bool FAST>
__device__ __forceinline__ float sigmoid_f32(float x) {
  return FAST ? rcp_fast(1.f + __expf(-x)) : __frcp_rn(1.f + exp_f32(-x));
}

// act(x) and act'(x):
//   silu       x s,        s (1 + x (1 - s)),               s = sigmoid(x)
//   gelu       x Phi(x),   Phi(x) + x phi(x)                (normal distribution function and density)
//   gelu_tanh  x s,        s (1 + x (1 - s) 2 w'),          s = sigmoid(2 w) = (1 + tanh w) / 2,  w = sqrt(2/pi) (x + 0.044715 x^3)
template <int ACT, bool FAST>
__device__ __forceinline__ void act_and_derivative(float x, float& act, float& der) {
  if (ACT == ACT_GELU && FAST) {
    // Abramowitz and Stegun 7.1.26, erfc(z) = (a1 t + ... + a5 t^5) e^-z^2 with t = 1 / (1 + p z), off by at most 1.5e-7; the
    // exponential is the density's too (8192 x 8192 values in bf16: 76 us forward and 114 backward, 93 and 131 with erff)
    const float e = __expf(-0.5f * x * x), t = rcp_fast(fmaf(0.3275911f * 0.707106781f, fabsf(x), 1.f));
    const float tail = 0.5f * e * t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f);
    const float cdf = x < 0.f ? tail : 1.f - tail;
    act = x * cdf;
    der = fmaf(x, 0.398942280f * e, cdf);
  } else if (ACT == ACT_GELU) {
    const float cdf = 0.5f * erfcf(-0.707106781f * x);
    act = x * cdf;
    der = fmaf(x, 0.398942280f * exp_f32(-0.5f * x * x), cdf);
  } else {
    const float k = 1.59576912f, c = 0.044715f;   // 2 sqrt(2/pi)
    const float s = sigmoid_f32<FAST>(ACT == ACT_SILU ? x : k * x * fmaf(c * x, x, 1.f));
    const float slope = ACT == ACT_SILU ? 1.f : k * fmaf(3.f * c * x, x, 1.f);
    act = x * s;
    der = s * fmaf(x * (1.f - s), slope, 1.f);
  }
}

template <int ACT, bool FAST>
__device__ __forceinline__ float activation(float x) {
  float act, der;
  act_and_derivative<ACT, FAST>(x, act, der);
  return act;
}

}  // namespace sb
