// Activations of the linear with an epilogue, and their derivatives: FP32, the library's accurate erf / tanh / exp.
// Codes as RTXB_ACT_*.
#pragma once

#include "common.cuh"

namespace rtxb {

enum Activation : int { kActNone = 0, kActRelu = 1, kActRelu2 = 2, kActSilu = 3, kActGelu = 4, kActGeluTanh = 5 };

constexpr float kSqrtHalf = 0.70710678118654752f;
constexpr float kInvSqrt2Pi = 0.39894228040143268f;
constexpr float kGeluTanhA = 0.79788456080286536f;   // sqrt(2 / pi)
constexpr float kGeluTanhB = 0.044715f;

// Beyond +-128 silu and the two gelus are their limits to the last bit (e^128 overflows, erf and tanh are +-1), so the
// arguments are held there: infinities and the type's lowest value give the limit (0, z, slope 0 or 1) and not inf * 0.
// NaN passes through (the comparisons are false).
template <int ACT>
__device__ __forceinline__ float act_value(float z) {
  if (ACT == kActRelu) return z < 0.0f ? 0.0f : z;
  if (ACT == kActRelu2) return z < 0.0f ? 0.0f : z * z;
  if (ACT != kActNone) z = z < -128.0f ? -128.0f : z;
  if (ACT == kActSilu) return z / (1.0f + expf(-z));
  if (ACT == kActGelu) return 0.5f * z * (1.0f + erff(z * kSqrtHalf));
  if (ACT == kActGeluTanh) return 0.5f * z * (1.0f + tanhf(kGeluTanhA * (z + kGeluTanhB * z * z * z)));
  return z;
}

// act'(z); relu has slope 0 at 0
template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
  if (ACT == kActRelu) return z > 0.0f ? 1.0f : (z == z ? 0.0f : z);
  if (ACT == kActRelu2) return z > 0.0f ? 2.0f * z : (z == z ? 0.0f : z);
  z = z < -128.0f ? -128.0f : z > 128.0f ? 128.0f : z;
  if (ACT == kActSilu) {
    const float s = 1.0f / (1.0f + expf(-z));
    return s * (1.0f + z * (1.0f - s));
  }
  if (ACT == kActGelu) return 0.5f * (1.0f + erff(z * kSqrtHalf)) + z * kInvSqrt2Pi * expf(-0.5f * z * z);
  if (ACT == kActGeluTanh) {
    const float t = tanhf(kGeluTanhA * (z + kGeluTanhB * z * z * z));
    return 0.5f * (1.0f + t) + 0.5f * z * (1.0f - t * t) * kGeluTanhA * (1.0f + 3.0f * kGeluTanhB * z * z);
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
