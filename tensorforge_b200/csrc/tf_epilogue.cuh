// tf_epilogue.cuh -- what the linear layer's kernels do with an accumulated value:
//   z = acc * a_scale[m] * b_scale[n] + bias[n];  out = act(z) + residual[m, n]
// and the activations' derivatives for the gradient.  All in f32.
#pragma once
#include <cuda_bf16.h>

#include <type_traits>

#include "tf_internal.h"
#include "tf_ptx.cuh"

namespace tf {

// z / (1 + exp(-u)), the logistic gate: silu with u = z, the tanh form of gelu with
// u = 2 sqrt(2/pi) (z + 0.044715 z^3), since (1 + tanh a) / 2 = 1 / (1 + exp(-2 a)).  Where exp
// overflows the gate is 0, and __fdividef by a divisor above 2^126 gives that 0.  As in the formula,
// z = -inf gives NaN.
__device__ __forceinline__ float gated(float z, float u) { return __fdividef(z, 1.0f + __expf(-u)); }
constexpr float kGeluC = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float kGeluC3 = 0.044715f * kGeluC;

// z Phi(z), Phi(z) = (1 + erf(z / sqrt 2)) / 2: the sum cancels below z = -3, where the result's
// absolute error stays under 2^-24 |z|.
__device__ __forceinline__ float normal_cdf(float z) { return fmaf(0.5f, erff(z * 0.70710678118654752f), 0.5f); }

template <int ACT>
__device__ __forceinline__ float activate(float z) {
  if constexpr (ACT == TFORGE_ACT_RELU) return relu_ieee(z);
  else if constexpr (ACT == TFORGE_ACT_GELU) return z * normal_cdf(z);
  else if constexpr (ACT == TFORGE_ACT_GELU_TANH) return gated(z, z * fmaf(kGeluC3, z * z, kGeluC));
  else if constexpr (ACT == TFORGE_ACT_SILU) return gated(z, z);
  else return z;
}

// d act(z) / dz; at 0 the rectifier's is 0.
template <int ACT>
__device__ __forceinline__ float activate_slope(float z) {
  if constexpr (ACT == TFORGE_ACT_RELU) return z > 0.0f ? 1.0f : (z <= 0.0f ? 0.0f : z);
  else if constexpr (ACT == TFORGE_ACT_GELU)
    return fmaf(z, 0.3989422804014327f * __expf(-0.5f * z * z), normal_cdf(z));
  else if constexpr (ACT == TFORGE_ACT_GELU_TANH || ACT == TFORGE_ACT_SILU) {
    // s = 1 / (1 + exp(-u)): d(z s)/dz = s + z u' s (1 - s).
    constexpr bool kTanh = ACT == TFORGE_ACT_GELU_TANH;
    const float z2 = z * z;
    const float u = kTanh ? z * fmaf(kGeluC3, z2, kGeluC) : z;
    const float du = kTanh ? fmaf(3.0f * kGeluC3, z2, kGeluC) : 1.0f;
    const float s = __fdividef(1.0f, 1.0f + __expf(-u));
    const float v = s * (1.0f - s);
    return v == 0.0f ? s : fmaf(z * du, v, s);  // the gate is 0 or 1: z u' may have overflowed
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
