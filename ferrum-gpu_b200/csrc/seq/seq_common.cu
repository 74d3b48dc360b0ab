#include "seq_common.cuh"

namespace ferrum {
namespace seq {

namespace {
// 32 columns by 8 strands of rows; the strands' sums are added in order. The
// first `split` columns go to `out`, the others to `rest`.
__global__ void __launch_bounds__(256)
sum_rows_kernel(const float* __restrict__ part, int64_t rows, int64_t n, int64_t split,
                float* __restrict__ out, float* __restrict__ rest) {
  __shared__ float sh[8][32];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int64_t i = (int64_t)blockIdx.x * 32 + x;
  float s = 0.f;
  if (i < n) {
#pragma unroll 4
    for (int64_t r = y; r < rows; r += 8) s += part[r * n + i];
  }
  sh[y][x] = s;
  __syncthreads();
  if (y == 0 && i < n) {
#pragma unroll
    for (int k = 1; k < 8; ++k) s += sh[k][x];
    if (i < split)
      out[i] = s;
    else if (rest)
      rest[i - split] = s;
  }
}
}  // namespace

cudaError_t launch_sum_rows(const float* part, int64_t rows, int64_t n, int64_t split, float* out,
                            float* rest, cudaStream_t stream) {
  launch_detail::clear_stale_error();
  sum_rows_kernel<<<(unsigned)ceil_div(n, 32), 256, 0, stream>>>(part, rows, n, split, out, rest);
  return cudaGetLastError();
}

}  // namespace seq
}  // namespace ferrum
