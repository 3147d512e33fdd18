// Activations of the linear with an epilogue, and their derivatives, in FP32.  Codes as RTXB_ACT_*.
//
// The epilogue evaluates one activation per output element beside the MMAs of the next tile, so an evaluation may cost two
// special-function operations and some twenty multiply-adds; the library's erff / tanhf / expf cost two to four times that.
// Forms without cancellation:
//   silu       z s(z), s(z) = 1 / (1 + e^-z)
//   gelu_tanh  z s(2 a (z + b z^3)), since (1 + tanh u) / 2 = s(2 u)
//   gelu       z Phi(z) = max(z, 0) - |z| Phi(-|z|), Phi(-a) = e^(-a^2 / 2) (c1 t + .. + c7 t^7), t = 1 / (1 + p a)
// The polynomial is a minimax fit to Phi(-a) e^(a^2 / 2) on 0 <= a <= 14 in RELATIVE error, made for this file (8.1e-7 with
// the coefficients rounded to FP32), so that the far tail keeps as many digits as the rest: a fit with an absolute bound of
// 1e-7 is off by 1 % of gelu at z = -8.  Exponential and reciprocal are the hardware's (errors of a few 2^-23).  The
// exponent's roundings are 2^-24 of it each, so the relative error grows to 2^-16 where the power leaves the normal range,
// against the 2^-8 of the BF16 result's half step.  Results below 2^-119 in magnitude may come out as zero: s(z) or the
// power is then below 2^-126, and |z| below 88 (silu), 11 (gelu_tanh) or 14 (gelu).
#pragma once

#include "common.cuh"

namespace rtxb {

enum Activation : int { kActNone = 0, kActRelu = 1, kActRelu2 = 2, kActSilu = 3, kActGelu = 4, kActGeluTanh = 5 };

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
// -Phi(-a) for a >= 0.  The sign is in the coefficients.
__device__ __forceinline__ f32x2 minus_tail2(f32x2 a) {
  const f32x2 t = rcp2(fma2(a, both(0.362f), both(1.0f)));
  const f32x2 e = exp2_2(mul2(mul2(a, a), both(-0.5f * kLog2E)));
  f32x2 c = fma2(t, both(-0.0479379926f), both(0.180008766f));
  c = fma2(c, t, both(-0.176616161f));
  c = fma2(c, t, both(-0.0288321568f));
  c = fma2(c, t, both(-0.139429476f));
  c = fma2(c, t, both(-0.142689345f));
  c = fma2(c, t, both(-0.144503904f));
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
    const f32x2 a = pack2(abs_upto_128(x), abs_upto_128(y));
    r = fma2(a, minus_tail2(a), pack2(fmax_nan(x, 0.0f), fmax_nan(y, 0.0f)));
  } else {
    const f32x2 z = pack2(fmax_nan(x, -128.0f), fmax_nan(y, -128.0f));
    r = mul2(z, ACT == kActSilu ? sigmoid2(z) : gelu_tanh_gate2(z, mul2(z, z)));
  }
  x = lo(r);
  y = hi(r);
}

// g * act'(z) of relu and relu2 for a pair; relu has slope 0 at 0
template <int ACT>
__device__ __forceinline__ void relu_slope2(float& gx, float& gy, float x, float y) {
  static_assert(ACT == kActRelu || ACT == kActRelu2, "the others are looked up");
  const float k = ACT == kActRelu ? 1.0f : 2.0f;
  gx *= x > 0.0f ? (ACT == kActRelu ? k : k * x) : (x == x ? 0.0f : x);
  gy *= y > 0.0f ? (ACT == kActRelu ? k : k * y) : (y == y ? 0.0f : y);
}

// act'(-a), 0 <= a <= 128, of silu and the two gelus: the entries of the backward's table, a few thousand per block, so they
// are made to FP32 accuracy (a few 2^-24 of the slope, also beside its zero).  A slope that is off by 3e-7 moves dz across a
// BF16 rounding, and now and then an E4M3 code behind it, for every gradient of an unlucky z: in the training step of
// 8192 x 4096 x 8192 that was 2.1e-4 of dx (2-norm), where the MMAs' accumulation is 1.2e-4 and these entries are 0.
//   silu, gelu_tanh  with s(-u) = q / (1 + q), q = e^-u:   q (1 - a u'(a) + q) / (1 + q)^2;  u = a,  or 2 A (a + B a^3)
//   gelu             Phi(-a) - a phi(a) = e^(-a^2 / 2) (a0 - a) h(a): a0 its zero, in two parts, h a polynomial in
//                    1 / (1 + 0.32 a) fitted as above on 0 <= a <= 14 (4.6e-8)
// The exponents are formed in FP64 and their rounding to FP32 is put back into the power.
__device__ __forceinline__ float exp2_of(double x) {   // x <= 0
  const float head = static_cast<float>(x);
  float p;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p) : "f"(head));
  return fmaf(p, static_cast<float>(x - head) * 0.693147181f, p);
}
__device__ __forceinline__ float slope_at_minus(int act, float a) {
  constexpr double kLog2 = 1.4426950408889634, kA = 0.79788456080286536, kB = 0.044715;
  const double d = a;
  if (act == kActGelu) {
    const float t = 1.0f / fmaf(a, 0.32f, 1.0f);
    float h = fmaf(t, 0.0130718084f, -0.0584661273f);
    h = fmaf(h, t, 0.0741537535f);
    h = fmaf(h, t, -0.00356778049f);
    h = fmaf(h, t, 0.0692133608f);
    h = fmaf(h, t, 0.075452407f);
    h = fmaf(h, t, 0.0962936944f);
    h = fmaf(h, t, 0.398926866f);
    return exp2_of(-0.5 * kLog2 * d * d) * ((0.751791537f - a) - 1.21144495e-08f) * h;
  }
  const bool silu = act == kActSilu;
  const double u = silu ? d : 2.0 * kA * d * (1.0 + kB * d * d), slope = silu ? 1.0 : 2.0 * kA * (1.0 + 3.0 * kB * d * d);
  const float q = exp2_of(-kLog2 * u), r = 1.0f / (1.0f + q);
  return q * (static_cast<float>(1.0 - d * slope) + q) * r * r;
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
