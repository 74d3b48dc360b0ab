// Softmax cross entropy against a vocabulary matrix: what its translation
// units share.
#pragma once

#include "seq_common.cuh"

namespace ferrum {
namespace seq {

struct LossSizes {
  int64_t tokens, width, vocab;
};

__device__ __forceinline__ bool has_loss(int64_t target, int64_t vocab) {
  return target >= 0 && target < vocab;
}

// Largest value and the sum of e^(value - largest) of some of a row's logits.
// Where the largest is infinite, the sum is of e^value.
struct RowStat {
  float top, sum;
};
__device__ __forceinline__ float shift_of(float top) { return fabsf(top) == INFINITY ? 0.f : top; }
__device__ __forceinline__ RowStat join(RowStat a, RowStat b) {
  RowStat r;
  r.top = fmaxf(a.top, b.top);
  const float s = shift_of(r.top);
  const float wa = a.top == -INFINITY ? 0.f : ex2((shift_of(a.top) - s) * kLog2e);
  const float wb = b.top == -INFINITY ? 0.f : ex2((shift_of(b.top) - s) * kLog2e);
  r.sum = a.sum * wa + b.sum * wb;
  return r;
}

__device__ __forceinline__ float lse_of(RowStat r) { return shift_of(r.top) + logf(r.sum); }

ferrum_status loss_fwd_f32(ferrum_device* dev, const ferrum_cross_entropy_args* a,
                           cudaStream_t stream, const char* what);
ferrum_status loss_bwd_f32(ferrum_device* dev, const ferrum_cross_entropy_args* a,
                           cudaStream_t stream, const char* what);
ferrum_status loss_fwd_tc(ferrum_device* dev, const ferrum_cross_entropy_args* a,
                          cudaStream_t stream, const char* what);
ferrum_status loss_bwd_tc(ferrum_device* dev, const ferrum_cross_entropy_args* a,
                          cudaStream_t stream, const char* what);

}  // namespace seq
}  // namespace ferrum
