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
// part in 2^22), Phi(-x) = exp(-x^2/2) t Q(t) with t = 1 / (1 + 0.43 x / sqrt(2)) and a polynomial Q of degree seven that
// was fitted to exp(y^2) erfc(y) / 2t, y = x / sqrt(2), on 0 .. 9.5 for the smallest largest relative error (weighted least
// squares with weights that follow the error): 8.4e-8 = 2^-23.5; with the rounded argument of the exponential 4e-7 up to
// x = 2, 1.4e-6 up to 5, against 4.9e-4 of an fp16 result's rounding (degree five: 5.2e-6, and one result in 200 rounded
// the wrong way). The two products more than degree five cost 8192 x 8192 x 4096 with GELU and Z 468 -> 471 us, nothing where
// memory or another rate is the bound: GELU's gradient of 8192 x 8192 with the bias's 78.3 -> 78.0 us, 4096 x 8192 x 2048 through
// it 140.9 -> 140.3 (a clamp stands where a comparison and a selection stood). Tried on a card where the former takes 473.1
// with degree five and 477.7 with seven: degree six (7.4e-7) 476.2, two halves of the polynomial side by side 480.2; a
// polynomial of degree seven without the factor t (2.5e-7) saves a product and no time, with 2.5 times as many results rounded the
// wrong way. The other form, for fp32 results, calls the math library.
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
    bell = __builtin_amdgcn_exp2f(-0.72134752f * (z * z));  // -log2(e) / 2; z^2 of a 16-bit z is exact
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.43f * 0.70710678f, __builtin_fabsf(z), 1.0f));
    float q = __builtin_fmaf(0.0368538201f, t, -0.155186132f);
    q = __builtin_fmaf(q, t, 0.191851914f);
    q = __builtin_fmaf(q, t, -0.0428620428f);
    q = __builtin_fmaf(q, t, 0.123421796f);
    q = __builtin_fmaf(q, t, 0.102475673f);
    q = __builtin_fmaf(q, t, 0.122187704f);
    q = __builtin_fmaf(q, t, 0.121257305f);
    return q * t * bell;
  } else {
    bell = expf(-0.5f * z * z);
    return 0.5f * erfcf(0.70710678f * __builtin_fabsf(z));
  }
}

// z, or zero where the factor that it meets is zero: an infinite z (a Z that overflowed 16 bits) has its limits, not infinity
// times zero. A NaN comes in through that factor.
__device__ __forceinline__ float Meeting(const float z, const float factor) { return (factor > 0.0f) ? z : 0.0f; }

// Beyond it the bell and the tail of the normal distribution are zero in 32 bits: a z that is held inside brings no infinity times zero
constexpr float kGeluEnd = 20.0f;

constexpr float kTanhSlope = 0.79788456f;  // sqrt(2 / pi)

// act(z). `activation` is the same for the whole launch.
template <bool FAST>
__device__ __forceinline__ float Activate(const int activation, const float z) {
  switch (activation) {
    case kActivationRelu: return (z < 0.0f) ? 0.0f : z;  // (a NaN stays one)
    case kActivationGelu: {  // z Phi(z): z - z Phi(-z) on the positive side, z Phi(-|z|) on the other
      float bell;
      const float tail = NormalTail<FAST>(z, bell);
      const float c = __builtin_amdgcn_fmed3f(z, -kGeluEnd, kGeluEnd);  // (a NaN comes in through the tail)
      return __builtin_fmaf(-__builtin_fabsf(c), tail, (z < 0.0f) ? 0.0f : z);
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
      const float c = __builtin_amdgcn_fmed3f(z, -kGeluEnd, kGeluEnd);  // (a NaN comes in through the bell)
      return __builtin_fmaf(0.39894228f * c, bell, (z > 0.0f) ? 1.0f - tail : tail);  // 1 / sqrt(2 pi)
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
