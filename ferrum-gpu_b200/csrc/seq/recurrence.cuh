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

// sigmoid(x) and 1 - sigmoid(x), each with a relative error of a few units: the
// smaller one is e / (1 + e) with e = e^-|x|, and is kept (its sign set for x > 0).
struct Gate {
  float small;
  __device__ __forceinline__ bool open() const { return __float_as_int(small) < 0; }
  __device__ __forceinline__ float on() const { return open() ? 1.f + small : small; }
  __device__ __forceinline__ float off() const { return open() ? -small : 1.f - small; }
};
__device__ __forceinline__ Gate gate_of(float x) {
  const float e = ex2(-fabsf(x) * kLog2e);
  const float t = e * rcp(1.f + e);
  return {x > 0.f ? -t : t};
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
  // a h + b, the sum of the small terms first
  __device__ __forceinline__ float step(float h, float b) const {
    return fmaf(code, h, b) + rest(h);
  }
};
constexpr float kKeep = -0.f;                   // the code of a = 1

// e^x for x <= 88: x = k ln 2 + r with |r| <= ln 2 / 2; (e^r - 1 - r) / r^2 by a
// polynomial of degree 4, fitted for the relative error of e^r - 1 (largest 0.23
// units of 2^-24). One rounded ln 2 is enough: k of it shifts e^r by k 2e-9, of an
// a that is 2^k. Below -87 the factor is 0; NaN stays NaN.
// `w`: 1 - a^2 with its relative accuracy.
__device__ __forceinline__ Factor factor_of(float x, float* w = nullptr) {
  const float magic = 12582912.f;                    // 1.5 * 2^23: rounds to an integer
  float v = x < -87.f ? -87.f : x;
  v = v > 88.f ? 88.f : v;
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
  const bool near = k == 0.f && v <= 0.f;
  if (w) *w = near ? -q * (2.f + q) : fmaf(-a, a, 1.f);
  return {near ? -fabsf(q) : a};
}

struct Decay {
  Factor a;
  float inv, w;       // 1 / sqrt(w) with w = 1 - a^2; 0 where that is not above 2^-126
  __device__ __forceinline__ float root() const { return w * inv; }
};
__device__ __forceinline__ Decay decay_of(float decay, float r) {
  Decay d;
  d.a = factor_of(-decay * r, &d.w);
  float s;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(d.w));
  d.inv = d.w > 1.1754944e-38f ? s : 0.f;
  return d;
}

// What a step adds to the gradients, from the state's gradient g, the state in
// front of the step, x and the gates.
struct StepGrads {
  float dx, dig, drg, ddecay;
};
__device__ __forceinline__ StepGrads step_grads(float g, float before, float x, Gate i, Gate r,
                                                const Decay& d, float decay) {
  StepGrads s;
  s.dx = g * d.root() * i.on();
  s.dig = s.dx * x * i.off();
  // d(a)/d(la) = a, d(root)/d(la) = -a^2 / root
  const float a = d.a.value();
  const float dla = g * a * fmaf(-a * d.inv, i.on() * x, before);
  s.ddecay = -r.on() * dla;
  s.drg = s.ddecay * decay * r.off();
  return s;
}

}  // namespace seq
}  // namespace ferrum
