// Activations and their derivatives of the training-step kernels (norm.hip, gated.hip), in FP32.
#pragma once

#include <type_traits>

#include "common.h"

namespace fim {

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3, ACT_GELU_TANH = 4, ACT_COUNT = 5 };

// The normal distribution's upper tail E(|z|) = erfc(|z| / sqrt 2) / 2 as 2^P(|z|), P a degree-10 fit of log2 E on
// [0, 5.6] (this repository's own; 5e-8 absolute in E with FP32 Horner steps, which in powers of |z| itself start with no
// cancellation). Its leading coefficient is negative: past the fit E falls to 0, at infinity too. Three FMAs more than
// gelu_erf's fit: FP32 outputs and parameter gradients are held to 1e-6 here, where that one's 3e-6 showed.
__device__ __forceinline__ float normal_tail(float az) {
  constexpr float c[10] = {7.012681066953519e-07f, -9.234423487214372e-06f, 6.613872392335907e-05f,
                           -0.00024351512547582388f, -7.589748565806076e-05f, 0.007040276657789946f,
                           -0.05250448361039162f, -0.45920008420944214f, -1.1511067152023315f, -0.9999999403953552f};
  float p = -2.28585239625545e-08f;
#pragma unroll
  for (int k = 0; k < 10; ++k) p = fmaf(p, az, c[k]);
  return __builtin_amdgcn_exp2f(p);
}

// 1 / (1 + e^-z); 0 and 1 at the infinities
__device__ __forceinline__ float logistic(float z) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504088896341f * z));
}

constexpr float kTanhA = 0.79788456080286535588f;  // sqrt(2 / pi)
constexpr float kTanhB = 0.044715f;

// act(z), and act'(z) in `slope` where WITH_SLOPE, as autograd has them: ReLU's slope is 0 at 0 and 1 at NaN, the others' NaN.
//   SiLU: z s, s (1 + z (1 - s)) with s = logistic(z)
//   GELU: z Phi(z) = max(z, 0) - |z| E, Phi(z) + z phi(z)
//   GELU, tanh form: z s with s = logistic(2 y), y = a (z + b z^3) (0.5 (1 + tanh y) = s); s + z s (1 - s) 2 y'
template <int ACT, bool WITH_SLOPE>
__device__ __forceinline__ float activate(float z, float& slope) {
  if constexpr (ACT == ACT_NONE) {
    if constexpr (WITH_SLOPE) slope = 1.0f;
    return z;
  } else if constexpr (ACT == ACT_RELU) {
    if constexpr (WITH_SLOPE) slope = z <= 0.0f ? 0.0f : 1.0f;
    return __builtin_elementwise_maximum(z, 0.0f);  // NaN stays NaN
  } else if constexpr (ACT == ACT_SILU) {
    const float s = logistic(z);
    if constexpr (WITH_SLOPE) slope = s * fmaf(z, 1.0f - s, 1.0f);
    return z * s;
  } else if constexpr (ACT == ACT_GELU) {
    const float az = fabsf(z), e = normal_tail(az);
    if constexpr (WITH_SLOPE) {
      const float pdf = 0.39894228040143267794f * __builtin_amdgcn_exp2f(-0.72134752044448170368f * z * z);
      slope = fmaf(__builtin_amdgcn_fmed3f(z, -3e38f, 3e38f), pdf, z > 0.0f ? 1.0f - e : e);
    }
    return fmaf(-__builtin_elementwise_minimum(az, 3e38f), e, __builtin_elementwise_maximum(z, -0.0f));
  } else {
    // s is 0 or 1 long before the bounds: no inf times 0 (minimum and maximum keep a NaN, the median would not)
    const float zc = __builtin_elementwise_minimum(__builtin_elementwise_maximum(z, -1e4f), 1e4f), z2 = zc * zc;
    const float s = logistic(2.0f * kTanhA * zc * fmaf(kTanhB, z2, 1.0f));
    if constexpr (WITH_SLOPE) slope = s * fmaf(zc * (1.0f - s), 2.0f * kTanhA * fmaf(3.0f * kTanhB, z2, 1.0f), 1.0f);
    return z * s;
  }
}

template <int ACT>
__device__ __forceinline__ float activate(float z) {
  float unused;
  return activate<ACT, false>(z, unused);
}

// f(std::integral_constant<int, ACT>) for the runtime code `act`, which the caller has checked
template <typename F>
inline void with_activation(int act, F&& f) {
  switch (act) {
    case ACT_NONE: f(std::integral_constant<int, ACT_NONE>{}); break;
    case ACT_RELU: f(std::integral_constant<int, ACT_RELU>{}); break;
    case ACT_SILU: f(std::integral_constant<int, ACT_SILU>{}); break;
    case ACT_GELU: f(std::integral_constant<int, ACT_GELU>{}); break;
    default: f(std::integral_constant<int, ACT_GELU_TANH>{}); break;
  }
}

}  // namespace fim
