// =================================================================================================
// The activations of the layer products (kernels/layer_gemm.hpp) and their derivatives, on fp32 values:
//   relu       max(z, 0)
//   gelu       z Phi(z), Phi the normal distribution function
//   gelu_tanh  z / (1 + exp(-2u)) with u = sqrt(2/pi) (z + 0.044715 z^3)   (the tanh form: (1 + tanh u) / 2 = 1 / (1 + exp(-2u)))
//   silu       z / (1 + exp(-z))
// Written so that the small values on the negative side keep their relative accuracy: no 1 + erf or 1 + tanh, whose
// cancellation leaves nothing of Phi(-5).
//
// Two forms. FAST, for results that are rounded to 16 bits: the exponential and the reciprocal of the hardware (about one
// part in 2^22), Phi(-x) = exp(-x^2/2) Q(t) / 2 with t = 1 / (1 + 0.43 x / sqrt(2)) and a polynomial Q of degree six that
// was fitted to exp(y^2) erfc(y), y = x / sqrt(2), on 0 .. 9.5 for the smallest largest relative error (weighted least
// squares with weights that follow the error): 5.2e-6 = 2^-17.6, against 2^-12 of an fp16 result's rounding; beyond, where
// exp(-y^2) is less than 1e-39, 5e-5. The other form, for fp32 results, calls the math library.
// =================================================================================================
#ifndef CLBLAST_HIP_KERNELS_ACTIVATIONS_HPP_
#define CLBLAST_HIP_KERNELS_ACTIVATIONS_HPP_

#include <hip/hip_runtime.h>

namespace clbh {

// The values of CLBlastActivation (include/clblast_hip_c.h)
constexpr int kActivationNone = 161, kActivationRelu = 162, kActivationGelu = 163, kActivationGeluTanh = 164,
              kActivationSilu = 165;

template <bool FAST>
__device__ __forceinline__ float Exponential(const float x) {
  return FAST ? __builtin_amdgcn_exp2f(x * 1.44269504f) : expf(x);
}
template <bool FAST>
__device__ __forceinline__ float Reciprocal(const float x) {
  return FAST ? __builtin_amdgcn_rcpf(x) : 1.0f / x;
}

// Phi(-|z|); `bell` receives exp(-z^2 / 2)
template <bool FAST>
__device__ __forceinline__ float NormalTail(const float z, float& bell) {
  if constexpr (FAST) {
    bell = __builtin_amdgcn_exp2f(-0.72134752f * z * z);  // -log2(e) / 2
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.43f * 0.70710678f, __builtin_fabsf(z), 1.0f));
    float q = __builtin_fmaf(0.5f * -0.15338767f, t, 0.5f * 0.40704837f);
    q = __builtin_fmaf(q, t, 0.5f * -0.01078906f);
    q = __builtin_fmaf(q, t, 0.5f * 0.28136584f);
    q = __builtin_fmaf(q, t, 0.5f * 0.23251006f);
    q = __builtin_fmaf(q, t, 0.5f * 0.24325760f);
    return q * t * bell;
  } else {
    bell = expf(-0.5f * z * z);
    return 0.5f * erfcf(0.70710678f * __builtin_fabsf(z));
  }
}

// z, or zero where the factor that it meets is zero: an infinite z (a Z that overflowed 16 bits) has its limits, not infinity
// times zero. A NaN comes in through that factor.
__device__ __forceinline__ float Meeting(const float z, const float factor) { return (factor > 0.0f) ? z : 0.0f; }

constexpr float kTanhSlope = 0.79788456f;  // sqrt(2 / pi)

// act(z). `activation` is the same for the whole launch.
template <bool FAST>
__device__ __forceinline__ float Activate(const int activation, const float z) {
  switch (activation) {
    case kActivationRelu: return (z < 0.0f) ? 0.0f : z;  // (a NaN stays one)
    case kActivationGelu: {  // z Phi(z): z - z Phi(-z) on the positive side, z Phi(-|z|) on the other
      float bell;
      const float tail = NormalTail<FAST>(z, bell);
      return __builtin_fmaf(-__builtin_fabsf(Meeting(z, tail)), tail, (z < 0.0f) ? 0.0f : z);  // (a NaN stays one)
    }
    case kActivationGeluTanh: {
      const float u = kTanhSlope * z * __builtin_fmaf(0.044715f * z, z, 1.0f);
      const float s = Reciprocal<FAST>(1.0f + Exponential<FAST>(-2.0f * u));
      return Meeting(z, s) * s;
    }
    case kActivationSilu: {
      const float s = Reciprocal<FAST>(1.0f + Exponential<FAST>(-z));
      return Meeting(z, s) * s;
    }
    default: return z;
  }
}

// act'(z)
template <bool FAST>
__device__ __forceinline__ float ActivationSlope(const int activation, const float z) {
  switch (activation) {
    case kActivationRelu: return (z > 0.0f) ? 1.0f : 0.0f;
    case kActivationGelu: {
      float bell;
      const float tail = NormalTail<FAST>(z, bell);
      return __builtin_fmaf(0.39894228f * Meeting(z, bell), bell, (z > 0.0f) ? 1.0f - tail : tail);  // 1 / sqrt(2 pi)
    }
    case kActivationGeluTanh: {
      const float u = kTanhSlope * z * __builtin_fmaf(0.044715f * z, z, 1.0f);
      // s = 1 / (1 + exp(-2u)), 1 - s = 1 / (1 + exp(2u)); the product of the two is the slope of s over 2u
      const float s = Reciprocal<FAST>(1.0f + Exponential<FAST>(-2.0f * u));
      const float r = Reciprocal<FAST>(1.0f + Exponential<FAST>(2.0f * u));
      // (s r is below 2^-126 beyond 20: clamped there, so that a huge z does not bring in infinity times zero)
      const float c = __builtin_fminf(__builtin_fmaxf(z, -20.0f), 20.0f);
      return s + 2.0f * kTanhSlope * c * __builtin_fmaf(3.0f * 0.044715f * c, c, 1.0f) * (s * r);
    }
    case kActivationSilu: {
      const float s = Reciprocal<FAST>(1.0f + Exponential<FAST>(-z));
      const float r = Reciprocal<FAST>(1.0f + Exponential<FAST>(z));
      return __builtin_fmaf(Meeting(z, s * r), s * r, s);
    }
    default: return 1.0f;
  }
}

}  // namespace clbh

#endif  // CLBLAST_HIP_KERNELS_ACTIVATIONS_HPP_
