// Arithmetic of one step of the gated recurrence, shared by its kernels:
//   r = sigmoid(rg), i = sigmoid(ig), la = -decay r, a = e^la,
//   root = sqrt(1 - a^2),  h = a h + root i x
// a lies close to 1 over long memories: a relative error of 2^-22, as the
// special-function unit's exponential has it, or the rounding of a itself under a
// gate that stands still, would add up over a thousand steps to 2e-4 or 3e-5 of the
// state. So where a > 0.7 its distance from 1 is kept, with a relative error of 1.5
// units of 2^-24, and the state moves by h + (a - 1) h; below, a h forgets a large
// state without leaving its rounding behind.
#pragma once

#include "seq_common.cuh"

namespace ferrum {
namespace seq {

// sigmoid(x) and 1 - sigmoid(x), each with a relative error of a few units; below -4 of |x|
// / 2 units more, from rounding the exponential's argument.
struct Gate {
  float on, off;
};
__device__ __forceinline__ Gate gate_of(float x) {
  const float e = ex2(-x * kLog2e), on = rcp(1.f + e);
  return {on, e < 3e38f ? e * on : 1.f};
}

// A factor a >= 0: a - 1 with the sign bit set, or a itself.
struct Factor {
  float code;
  __device__ __forceinline__ float rest(float h) const {    // h, or 0 where `code` is a
    return __int_as_float(__float_as_int(h) & (__float_as_int(code) >> 31));
  }
  __device__ __forceinline__ float value() const {
    return __float_as_int(code) < 0 ? 1.f + code : code;
  }
  __device__ __forceinline__ float times(float h) const { return fmaf(code, h, rest(h)); }
  // a h + b, the sum of the small terms first. An infinite h comes out as NaN, which
  // stays NaN in all steps to come; ANY keeps it infinite, as a > 0 does.
  template <bool ANY = false>
  __device__ __forceinline__ float step(float h, float b) const {
    return ANY && fabsf(h) == INFINITY ? h + b : fmaf(code, h, b) + rest(h);
  }
};
constexpr float kKeep = -0.f;                   // the code of a = 1

// A negative decay has no root: NaN.
__device__ __forceinline__ float checked_decay(float decay) { return decay < 0.f ? NAN : decay; }

// e^x for x <= 0: x = k ln 2 + r with |r| <= ln 2 / 2; (e^r - 1 - r) / r^2 by a
// polynomial of degree 4, fitted for the relative error of e^r - 1 (largest 0.30
// units of 2^-24, at r = -0.30). One rounded ln 2 is enough: k of it shifts e^r by k 2e-9, of an
// a that is 2^k. Below -87 the factor is 0; NaN stays NaN.
// `w`: 1 - a^2 with its relative accuracy.
__device__ __forceinline__ Factor factor_of(float x, float* w = nullptr) {
  const float magic = 12582912.f;                    // 1.5 * 2^23: rounds to an integer
  const float v = x < -87.f ? -87.f : x;
  const float kf = fmaf(v, kLog2e, magic);
  const float k = kf - magic;
  const float two_k = __int_as_float((__float_as_int(kf) << 23) + 0x3f800000);
  const float r = fmaf(k, -0.693147182464599609375f, v);
  float p = 0.0013946669641882181f;
  p = fmaf(p, r, 0.008366710506379604f);
  p = fmaf(p, r, 0.04166628047823906f);
  p = fmaf(p, r, 0.16666541993618011f);
  p = fmaf(p, r, 0.5f);
  const float q = fmaf(r * r, p, r);                 // e^r - 1
  const float a = x < -87.f ? 0.f : fmaf(two_k, q, two_k);
  const bool near = k == 0.f;
  if (w) *w = near ? -q * (2.f + q) : fmaf(-a, a, 1.f);
  return {near ? -fabsf(q) : a};
}

// e^x - 1 for x in [-1, 0], a polynomial as above, of degree 5 (largest relative error
// 0.17 units of 2^-24 before its own roundings, at x = -0.95): 8 instructions where factor_of takes 25.
constexpr float kShortDecay = 1.f;
__device__ __forceinline__ float expm1_short(float x) {
  float p = 0.00012913093087263405f;
  p = fmaf(p, x, 0.0013011264381930232f);
  p = fmaf(p, x, 0.00827620830386877f);
  p = fmaf(p, x, 0.04164746776223183f);
  p = fmaf(p, x, 0.16666366159915924f);
  p = fmaf(p, x, 0.49999985098838806f);
  return fmaf(x * x, p, x);
}

// sqrt(w) (w >= 0; 0 below 2^-126) and 1 / sqrt(w) (0 where w is not above 2^-126) to
// 2 units.
__device__ __forceinline__ float root_of(float w) {
  float s;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(w));
  return s;
}
__device__ __forceinline__ float inverse_root_of(float w) {
  float s;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(w));
  return w > 1.1754944e-38f ? s : 0.f;
}

// A step's factor and 1 - a^2. SHORT: decay lies in [0, kShortDecay], so a > 0.36
// and its distance from 1 serves throughout.
template <bool SHORT>
__device__ __forceinline__ Factor step_factor(float decay, float r, float& w) {
  if constexpr (SHORT) {
    const float m = expm1_short(-decay * r);
    w = -m * (2.f + m);
    return {m};
  } else {
    return factor_of(-decay * r, &w);
  }
}
template <bool SHORT>
__device__ __forceinline__ float step_times(Factor a, float h) {
  return SHORT ? fmaf(a.code, h, h) : a.times(h);
}
template <bool SHORT, bool ANY = false>
__device__ __forceinline__ float step_on(Factor a, float h, float b) {
  if (SHORT) return ANY && fabsf(h) == INFINITY ? h + b : fmaf(a.code, h, b) + h;
  return a.step<ANY>(h, b);
}

}  // namespace seq
}  // namespace ferrum
