// tf_epilogue.cuh -- what the linear layer's kernels do with an accumulated value:
//   z = acc * a_scale[m] * b_scale[n] + bias[n];  out = act(z) + residual[m, n]
// and the activations' derivatives for the gradient.  All in f32.
//
// The tensor core cuts where it adds to an f32 accumulator, so a sum over bf16 products shrinks by
// about 1.0e-6 of its value per 1024 of k (measured: 1.9e-5 at 16384; f32 additions that round leave
// 4e-7); e4m3's by 1.1e-6 at 16384.  That is lost in a bf16 output, not in an f32 one, whose sums are
// therefore taken in pieces -- of at most 768 (bf16) or 8192 (e4m3) -- and joined by rounding f32 additions:
// 7.4e-7 off at k = 4096 to 16384, and at worst 2^-24 of the sums for each piece joined.
#pragma once
#include <cuda_bf16.h>

#include <type_traits>

#include "tf_internal.h"
#include "tf_ptx.cuh"

namespace tf {

__device__ __forceinline__ float ex2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f;

// The logistic gate 1 / (1 + exp(-u)), u = -w / log2 e: silu is z gate(z), the tanh form of gelu
// z gate(2 sqrt(2/pi) (z + 0.044715 z^3)), since (1 + tanh a) / 2 = 1 / (1 + exp(-2 a)).  The factor
// -log2 e is folded into the polynomials.  Where 2^w overflows the gate is 0.
__device__ __forceinline__ float gate(float w) { return rcp_approx(1.0f + ex2_approx(w)); }
constexpr float kGeluC = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float kGeluC3 = 0.044715f * kGeluC;

// The normal distribution's Phi, and e = exp(-z^2 / 2), its density's shape.  The lower tail is
//   Phi(-x) = t q(t) exp(-x^2 / 2),  t = 1 / (1 + 0.305 x),
// with q of degree 7: the minimax fit, by linear programming, of the tail's relative error over 0 <= x <=
// 14 (8.5e-8), beyond where the exponential leaves f32.  With the roundings, half of them the
// exponent's, the tail is off by at most (9 + 0.75 z^2) 2^-23 of its value: 1e-6 near 0, 7e-6 at -8,
// where 1 + erf would have lost every digit.  Three steps more than a fit of the absolute error (1.5e-7,
// which is 5e-5 of the value at -3 and 1 % at -8).
__device__ __forceinline__ float normal_cdf(float z, float &e) {
  const float t = rcp_approx(fmaf(0.305f, fabsf(z), 1.0f));
  float q = fmaf(0.0365097337f, t, -0.152187902f);
  q = fmaf(q, t, 0.184324571f);
  q = fmaf(q, t, -0.0366914935f);
  q = fmaf(q, t, 0.120345789f);
  q = fmaf(q, t, 0.103622146f);
  q = fmaf(q, t, 0.122435505f);
  q = fmaf(q, t, 0.121641693f);
  e = ex2_approx(z * z * (-0.5f * kLog2e));
  const float tail = q * t * e;  // Phi(-|z|)
  return z > 0.0f ? 1.0f - tail : tail;
}

template <int ACT>
__device__ __forceinline__ float activate(float z) {
  if constexpr (ACT == TFORGE_ACT_RELU) return relu_ieee(z);
  else if constexpr (ACT == TFORGE_ACT_GELU) {
    float e;
    return z * normal_cdf(z, e);
  } else if constexpr (ACT == TFORGE_ACT_GELU_TANH) return z * gate(z * fmaf(-kLog2e * kGeluC3, z * z, -kLog2e * kGeluC));
  else if constexpr (ACT == TFORGE_ACT_SILU) return z * gate(-kLog2e * z);
  else return z;
}

// d act(z) / dz; at 0 the rectifier's is 0.
template <int ACT>
__device__ __forceinline__ float activate_slope(float z) {
  if constexpr (ACT == TFORGE_ACT_RELU) return z > 0.0f ? 1.0f : (z <= 0.0f ? 0.0f : z);
  else if constexpr (ACT == TFORGE_ACT_GELU) {
    float e;
    const float p = normal_cdf(z, e);
    return fmaf(z * 0.3989422804014327f, e, p);
  } else if constexpr (ACT == TFORGE_ACT_GELU_TANH || ACT == TFORGE_ACT_SILU) {
    // s = gate(u): d(z s)/dz = s + z u' s (1 - s).
    constexpr bool kTanh = ACT == TFORGE_ACT_GELU_TANH;
    const float z2 = z * z;
    const float w = kTanh ? z * fmaf(-kLog2e * kGeluC3, z2, -kLog2e * kGeluC) : -kLog2e * z;
    const float zdu = kTanh ? z * fmaf(3.0f * kGeluC3, z2, kGeluC) : z;
    const float s = gate(w);
    const float v = fmaf(-s, s, s);
    return v == 0.0f ? s : fmaf(zdu, v, s);  // the gate is 0 or 1: z u' may have overflowed
  } else return 1.0f;
}

// f(std::integral_constant<int, ACT>) for the run-time activation: one uniform branch around a loop.
template <typename F>
__device__ __forceinline__ void with_activation(int act, F &&f) {
  switch (act) {
    case TFORGE_ACT_RELU: f(std::integral_constant<int, TFORGE_ACT_RELU>()); break;
    case TFORGE_ACT_GELU: f(std::integral_constant<int, TFORGE_ACT_GELU>()); break;
    case TFORGE_ACT_GELU_TANH: f(std::integral_constant<int, TFORGE_ACT_GELU_TANH>()); break;
    case TFORGE_ACT_SILU: f(std::integral_constant<int, TFORGE_ACT_SILU>()); break;
    default: f(std::integral_constant<int, TFORGE_ACT_NONE>()); break;
  }
}

}  // namespace tf
