#include "seq_common.cuh"

namespace ferrum {
namespace seq {

namespace {
// 32 columns by 8 strands of rows; the strands' sums are added in order.
__global__ void __launch_bounds__(256)
sum_rows_kernel(const float* __restrict__ part, int64_t rows, int64_t n, int64_t row_stride,
                float* __restrict__ out) {
  __shared__ float sh[8][32];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int64_t i = (int64_t)blockIdx.x * 32 + x;
  float s = 0.f;
  if (i < n) {
#pragma unroll 4
    for (int64_t r = y; r < rows; r += 8) s += part[r * row_stride + i];
  }
  sh[y][x] = s;
  __syncthreads();
  if (y == 0 && i < n) {
#pragma unroll
    for (int k = 1; k < 8; ++k) s += sh[k][x];
    out[i] = s;
  }
}
}  // namespace

cudaError_t launch_sum_rows(const float* part, int64_t rows, int64_t n, int64_t row_stride,
                            float* out, cudaStream_t stream) {
  launch_detail::clear_stale_error();
  sum_rows_kernel<<<(unsigned)ceil_div(n, 32), 256, 0, stream>>>(part, rows, n, row_stride, out);
  return cudaGetLastError();
}

}  // namespace seq
}  // namespace ferrum
