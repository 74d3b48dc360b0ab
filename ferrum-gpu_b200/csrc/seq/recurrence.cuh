// Arithmetic of one step of the gated recurrence, shared by its kernels:
//   r = sigmoid(rg), i = sigmoid(ig), la = -decay r, a = e^la,
//   root = sqrt(1 - a^2),  h = a h + root i x
// a lies close to 1 over long memories: a relative error of 2^-22, as the
// special-function unit's exponential has it, would add up over a thousand
// steps to 2e-4 of the state. So m = e^la - 1 is computed on the FMA pipe with
// a relative error of 1.5 units of 2^-24, the state moves by h + m h, and
// 1 - a^2 = -m (2 + m) keeps its relative accuracy where a is close to 1.
#pragma once

#include "seq_common.cuh"

namespace ferrum {
namespace seq {

// e^x - 1 for x <= 88. x = k ln 2 + r with |r| <= ln 2 / 2; (e^r - 1 - r) / r^2
// by a polynomial of degree 4, fitted for the relative error of e^r - 1 (largest
// 0.23 units of 2^-24); then 2^k (e^r - 1) + (2^k - 1). One rounded ln 2 is
// enough: k of it shifts e^r by k 2e-9, of an a that is 2^k. Below -87 the
// result is -1; NaN stays NaN.
__device__ __forceinline__ float exp_m1(float x) {
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
  const float q = fmaf(r * r, p, r);
  const float m = fmaf(two_k, q, two_k - 1.f);
  return x < -87.f ? -1.f : m;
}

// sigmoid(x), and 1 - sigmoid(x) with a relative error that does not grow where
// sigmoid(x) rounds to 1.
struct Gate {
  float on, off;
};
__device__ __forceinline__ Gate gate_of(float x) {
  const float e = ex2(-x * kLog2e);
  Gate g;
  g.on = rcp(1.f + e);
  g.off = e < 3e38f ? e * g.on : 1.f;
  return g;
}

struct Decay {
  float m, a, inv, root;   // a - 1, a, 1 / sqrt(1 - a^2) (0 where that is not above 2^-126), sqrt
};
__device__ __forceinline__ Decay decay_of(float decay, float r) {
  Decay d;
  d.m = exp_m1(-decay * r);
  d.a = 1.f + d.m;
  const float w = -d.m * (1.f + d.a);
  float s;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(w));
  d.inv = w > 1.1754944e-38f ? s : 0.f;
  d.root = w * d.inv;
  return d;
}

// What a step adds to the gradients, from the state's gradient g, the state in
// front of the step, x and the gates.
struct StepGrads {
  float dx, dig, drg, ddecay;
};
__device__ __forceinline__ StepGrads step_grads(float g, float before, float x, Gate i, Gate r,
                                                Decay d, float decay) {
  StepGrads s;
  const float gi = g * d.root * i.on;
  s.dx = gi;
  s.dig = gi * x * i.off;
  // d(a)/d(la) = a, d(root)/d(la) = -a^2 / root
  const float dla = g * d.a * fmaf(-d.a * d.inv, i.on * x, before);
  s.ddecay = -r.on * dla;
  s.drg = s.ddecay * decay * r.off;
  return s;
}

}  // namespace seq
}  // namespace ferrum
