// Argument views and helpers shared by the selective scan's kernels.
#pragma once

#include "seq_common.cuh"

namespace ferrum {
namespace seq {

constexpr int kSaveSteps = FERRUM_SCAN_SAVE_STEPS;
constexpr float kLog2e = 1.4426950408889634f;

struct ScanSizes {
  int64_t batch, length, channels, groups, per_group, saves;
  int states;
  bool softplus;
};

template <class T>
struct ScanIn {
  Rows<T> u, delta, z, B, C;
  int64_t B_group, C_group;
  const float *A, *D, *bias;
  const float* initial;
  const int32_t* lengths;
};

__device__ __forceinline__ int64_t scan_length(const int32_t* lengths, int64_t b, int64_t length) {
  if (lengths == nullptr) return length;
  const int64_t n = lengths[b];
  return n < 0 ? 0 : (n > length ? length : n);
}

// 2^x by the special-function unit (2 units in the last place).
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// log(1 + e^x) = max(x, 0) + log(1 + e), e = e^-|x| in (0, 1]. log(1 + e) / e
// is a polynomial in e (least squares at Chebyshev nodes of [0, 1], relative
// error 3.1e-8), so small results keep their relative accuracy; it costs one
// exponential and ten products and sums, where log1pf takes a few times that
// and the scan spends it once per value.
__device__ __forceinline__ float softplus_f(float x) {
  const float e = ex2(-fabsf(x) * kLog2e);
  float p = 0.00525345793f;
  p = fmaf(p, e, -0.0295885075f);
  p = fmaf(p, e, 0.0783616677f);
  p = fmaf(p, e, -0.136747703f);
  p = fmaf(p, e, 0.191114306f);
  p = fmaf(p, e, -0.248443693f);
  p = fmaf(p, e, 0.333192706f);
  p = fmaf(p, e, -0.499995023f);
  p = fmaf(p, e, 1.f);
  return fmaf(p, e, fmaxf(x, 0.f));
}

// Pairs of floats for the two-wide FP32 instructions.
using f2 = unsigned long long;
__device__ __forceinline__ f2 pack(float x, float y) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 unpack(f2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

template <class T>
ScanIn<T> scan_in(const ferrum_scan_args* a) {
  return ScanIn<T>{rows_of<T>(a->u), rows_of<T>(a->delta), rows_of<T>(a->z), rows_of<T>(a->B),
                   rows_of<T>(a->C), a->B_group_stride, a->C_group_stride, a->A, a->D,
                   a->delta_bias, a->initial_state, a->lengths};
}

ferrum_status check_scan(const ferrum_device* dev, const ferrum_scan_args* a, const char* what,
                         bool bwd);

inline ScanSizes scan_sizes(const ferrum_scan_args* a) {
  ScanSizes s;
  s.batch = (int64_t)a->batch, s.length = (int64_t)a->length, s.channels = (int64_t)a->channels;
  s.groups = (int64_t)a->groups, s.per_group = s.channels / s.groups;
  s.saves = ceil_div(s.length, kSaveSteps);
  s.states = (int)a->states, s.softplus = a->delta_softplus != 0;
  return s;
}

template <class F>
ferrum_status with_states(int n, F f) {
  if (n <= 8) return f(std::integral_constant<int, 8>());
  if (n <= 16) return f(std::integral_constant<int, 16>());
  if (n <= 32) return f(std::integral_constant<int, 32>());
  return f(std::integral_constant<int, 64>());
}

}  // namespace seq
}  // namespace ferrum
