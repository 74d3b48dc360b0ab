#include "seq_common.cuh"

namespace ferrum {
namespace seq {

namespace {
__global__ void sum_rows_kernel(const float* __restrict__ part, int64_t rows, int64_t n,
                                float* __restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  float s = 0.f;
  for (int64_t r = 0; r < rows; ++r) s += part[r * n + i];
  out[i] = s;
}
}  // namespace

cudaError_t launch_sum_rows(const float* part, int64_t rows, int64_t n, float* out,
                            cudaStream_t stream) {
  launch_detail::clear_stale_error();
  sum_rows_kernel<<<(unsigned)ceil_div(n, 256), 256, 0, stream>>>(part, rows, n, out);
  return cudaGetLastError();
}

}  // namespace seq
}  // namespace ferrum
