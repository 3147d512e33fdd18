// Activations of the linear with an epilogue, and their derivatives, in FP32.  Codes as RTXB_ACT_*.
//
// The epilogue evaluates one activation per output element beside the MMAs of the next tile, the backward quantizer one
// slope per gradient element at memory speed, so an evaluation may cost two special-function operations and some twenty
// multiply-adds; the library's erff / tanhf / expf cost two to four times that.  Measured, gelu, 8192 x 8192: slope pass
// 210 us with erff and expf, 178 with the forms below a value at a time, 148 with them on packed pairs (and 110 with its
// table, quant_act.cuh); GEMM of 8192 x 4096 x 8192 with residual and z 265 us a value at a time, 217 on pairs.  Forms
// without cancellation:
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

// 1 / x and 2^x of both halves by the special-function unit
__device__ __forceinline__ f32x2 rcp2(f32x2 v) {
  float a, b;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(lo(v)));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(b) : "f"(hi(v)));
  return pack2(a, b);
}
__device__ __forceinline__ f32x2 exp2_2(f32x2 v) {
  float a, b;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(lo(v)));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(b) : "f"(hi(v)));
  return pack2(a, b);
}
constexpr float kLog2E = 1.4426950408889634f;

// s(z) for both; 0 and 1 at the ends (e^-z overflows to infinity, whose reciprocal is 0)
__device__ __forceinline__ f32x2 sigmoid2(f32x2 z) { return rcp2(add2(exp2_2(mul2(z, both(-kLog2E))), both(1.0f))); }
// s(2 a (z + b z^3)): the exponent is -2 a log2(e) z (1 + b z^2)
__device__ __forceinline__ f32x2 gelu_tanh_gate2(f32x2 z, f32x2 zz) {
  constexpr float k = -2.0f * kGeluTanhA * kLog2E;
  return rcp2(add2(exp2_2(mul2(z, fma2(zz, both(k * kGeluTanhB), both(k)))), both(1.0f)));
}
// -Phi(-a) for a >= 0; `e` receives e^(-a^2 / 2).  The 1/2 and the sign are in the coefficients.
__device__ __forceinline__ f32x2 minus_tail2(f32x2 a, f32x2& e) {
  const f32x2 t = rcp2(fma2(a, both(0.3275911f * kSqrtHalf), both(1.0f)));
  e = exp2_2(mul2(mul2(a, a), both(-0.5f * kLog2E)));
  f32x2 c = fma2(t, both(-0.5f * 1.061405429f), both(0.5f * 1.453152027f));
  c = fma2(c, t, both(-0.5f * 1.421413741f));
  c = fma2(c, t, both(0.5f * 0.284496736f));
  c = fma2(c, t, both(-0.5f * 0.254829592f));
  return mul2(c, mul2(t, e));
}
__device__ __forceinline__ float abs_upto_128(float z) { return fmin_nan(fabsf(z), 128.0f); }

// Beyond +-128 silu and the two gelus are their limits to the last bit (e^128 overflows, e^-8192 is 0), so what could
// become inf * 0 is held there: infinities and the type's lowest value give the limit (0, z, slope 0 or 1).  NaN passes
// through every step.
template <int ACT>
__device__ __forceinline__ void act_value2(float& x, float& y) {
  if (ACT == kActRelu || ACT == kActRelu2) {
    x = fmax_nan(x, 0.0f);
    y = fmax_nan(y, 0.0f);
    if (ACT == kActRelu2) { x *= x; y *= y; }
    return;
  }
  f32x2 r;
  if (ACT == kActGelu) {
    // z Phi(z) = max(z, 0) - |z| Phi(-|z|)
    f32x2 e;
    const f32x2 a = pack2(abs_upto_128(x), abs_upto_128(y));
    r = fma2(a, minus_tail2(a, e), pack2(fmax_nan(x, 0.0f), fmax_nan(y, 0.0f)));
  } else {
    const f32x2 z = pack2(fmax_nan(x, -128.0f), fmax_nan(y, -128.0f));
    r = mul2(z, ACT == kActSilu ? sigmoid2(z) : gelu_tanh_gate2(z, mul2(z, z)));
  }
  x = lo(r);
  y = hi(r);
}

// g * act'(z) for a pair; relu has slope 0 at 0
template <int ACT>
__device__ __forceinline__ void act_slope2(float& gx, float& gy, float x, float y) {
  if (ACT == kActRelu || ACT == kActRelu2) {
    const float k = ACT == kActRelu ? 1.0f : 2.0f;
    gx *= x > 0.0f ? (ACT == kActRelu ? k : k * x) : (x == x ? 0.0f : x);
    gy *= y > 0.0f ? (ACT == kActRelu ? k : k * y) : (y == y ? 0.0f : y);
    return;
  }
  const f32x2 one = both(1.0f);
  const f32x2 z = pack2(fmin_nan(fmax_nan(x, -128.0f), 128.0f), fmin_nan(fmax_nan(y, -128.0f), 128.0f));
  f32x2 d;
  if (ACT == kActSilu) {
    // s (1 + z (1 - s))
    const f32x2 s = sigmoid2(z);
    d = mul2(s, fma2(z, fma2(s, both(-1.0f), one), one));
  } else if (ACT == kActGelu) {
    // Phi(z) + z phi(z)
    f32x2 e;
    const f32x2 m = minus_tail2(pack2(fabsf(lo(z)), fabsf(hi(z))), e);
    const f32x2 up = add2(m, one);
    const f32x2 cdf = pack2(x < 0.0f ? -lo(m) : lo(up), y < 0.0f ? -hi(m) : hi(up));
    d = fma2(mul2(z, both(kInvSqrt2Pi)), e, cdf);
  } else {
    // s + z s (1 - s) 2 a (1 + 3 b z^2)
    const f32x2 zz = mul2(z, z);
    const f32x2 s = gelu_tanh_gate2(z, zz);
    const f32x2 w = mul2(mul2(z, s), fma2(zz, both(6.0f * kGeluTanhA * kGeluTanhB), both(2.0f * kGeluTanhA)));
    d = fma2(w, fma2(s, both(-1.0f), one), s);
  }
  d = mul2(pack2(gx, gy), d);
  gx = lo(d);
  gy = hi(d);
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
