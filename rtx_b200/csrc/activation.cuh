// Activations of the linear with an epilogue, and their derivatives, in FP32.  Codes as RTXB_ACT_*.
//
// The epilogue evaluates one activation per output element beside the MMAs of the next tile, the backward quantizer one
// slope per gradient element at memory speed, so an evaluation may cost two special-function operations and some twenty
// multiply-adds; the library's erff / tanhf / expf cost two to four times that (8192 x 4096 x 8192, gelu with z kept:
// the GEMM ran 315 us against 168 for the plain one, the slope pass 210 us at 30 % of the copy rate).  Forms without
// cancellation:
//   silu       z s(z), s(z) = 1 / (1 + e^-z)
//   gelu_tanh  z s(2 a (z + b z^3)), since (1 + tanh u) / 2 = s(2 u)
//   gelu       z Phi(z), Phi(-|z|) = erfc(|z| / sqrt 2) / 2 with erfc(x) = e^(-x^2) (c1 t + .. + c5 t^5), t = 1 / (1 + p x)
//              (Hastings' approximation, formula 7.1.26 of Abramowitz and Stegun, error below 1.5e-7), and
//              Phi(|z|) = 1 - Phi(-|z|)
// with the hardware exponential and reciprocal (relative errors of a few 2^-23 where the result is not negligible).
// The BF16 result's half step is 2^-8.
#pragma once

#include "common.cuh"

namespace rtxb {

enum Activation : int { kActNone = 0, kActRelu = 1, kActRelu2 = 2, kActSilu = 3, kActGelu = 4, kActGeluTanh = 5 };

constexpr float kSqrtHalf = 0.70710678118654752f;
constexpr float kInvSqrt2Pi = 0.39894228040143268f;
constexpr float kGeluTanhA = 0.79788456080286536f;   // sqrt(2 / pi)
constexpr float kGeluTanhB = 0.044715f;

__device__ __forceinline__ float fast_rcp(float x) {
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// 1 / (1 + e^-z): 0 and 1 at the ends (e^-z overflows to infinity, whose reciprocal is 0)
__device__ __forceinline__ float sigmoid(float z) { return fast_rcp(1.0f + __expf(-z)); }

// Phi(z); `e` receives e^(-z^2 / 2)
__device__ __forceinline__ float normal_cdf(float z, float& e) {
  const float x = fabsf(z) * kSqrtHalf;
  const float t = fast_rcp(fmaf(0.3275911f, x, 1.0f));
  e = __expf(-x * x);
  float c = fmaf(1.061405429f, t, -1.453152027f);
  c = fmaf(c, t, 1.421413741f);
  c = fmaf(c, t, -0.284496736f);
  c = fmaf(c, t, 0.254829592f);
  const float lower = 0.5f * c * t * e;
  return z < 0.0f ? lower : 1.0f - lower;
}

// Beyond +-128 silu and the two gelus are their limits to the last bit (e^128 overflows, e^-8192 is 0), so the arguments
// are held there: infinities and the type's lowest value give the limit (0, z, slope 0 or 1) and not inf * 0.
// NaN passes through (the comparisons are false).
template <int ACT>
__device__ __forceinline__ float act_value(float z) {
  if (ACT == kActRelu) return z < 0.0f ? 0.0f : z;
  if (ACT == kActRelu2) return z < 0.0f ? 0.0f : z * z;
  if (ACT != kActNone) z = z < -128.0f ? -128.0f : z;
  if (ACT == kActSilu) return z * sigmoid(z);
  if (ACT == kActGelu) {
    float e;
    return z * normal_cdf(z, e);
  }
  if (ACT == kActGeluTanh) return z * sigmoid(2.0f * kGeluTanhA * z * fmaf(kGeluTanhB * z, z, 1.0f));
  return z;
}

// act'(z); relu has slope 0 at 0
template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
  if (ACT == kActRelu) return z > 0.0f ? 1.0f : (z == z ? 0.0f : z);
  if (ACT == kActRelu2) return z > 0.0f ? 2.0f * z : (z == z ? 0.0f : z);
  z = z < -128.0f ? -128.0f : z > 128.0f ? 128.0f : z;
  if (ACT == kActSilu) {
    const float s = sigmoid(z);
    return s * fmaf(z, 1.0f - s, 1.0f);
  }
  if (ACT == kActGelu) {
    float e;
    const float cdf = normal_cdf(z, e);
    return fmaf(z * kInvSqrt2Pi, e, cdf);
  }
  if (ACT == kActGeluTanh) {
    // d(2u)/dz = 2 a (1 + 3 b z^2)
    const float s = sigmoid(2.0f * kGeluTanhA * z * fmaf(kGeluTanhB * z, z, 1.0f));
    return fmaf(z * s * (1.0f - s), 2.0f * kGeluTanhA * fmaf(3.0f * kGeluTanhB * z, z, 1.0f), s);
  }
  return 1.0f;
}

template <int ACT>
struct ActTag {
  static constexpr int value = ACT;
};

// f(tag) with the activation as a compile-time constant (not called for none): one branch per chunk of values
template <typename F>
__device__ __forceinline__ void with_activation(int act, F&& f) {
  switch (act) {
    case kActRelu: f(ActTag<kActRelu>{}); break;
    case kActRelu2: f(ActTag<kActRelu2>{}); break;
    case kActSilu: f(ActTag<kActSilu>{}); break;
    case kActGelu: f(ActTag<kActGelu>{}); break;
    case kActGeluTanh: f(ActTag<kActGeluTanh>{}); break;
    default: break;
  }
}

}  // namespace rtxb
