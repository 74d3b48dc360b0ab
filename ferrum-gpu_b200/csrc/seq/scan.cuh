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

// log(1 + e^x): x itself from 20 up (the difference, below e^-20, is lost to
// rounding there); log1pf keeps the relative accuracy where e^x is small.
__device__ __forceinline__ float softplus_f(float x) {
  return x > 20.f ? x : log1pf(__expf(x));
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
