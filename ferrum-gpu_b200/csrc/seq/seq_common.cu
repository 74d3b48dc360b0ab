#include "seq_common.cuh"

namespace ferrum {
namespace seq {

namespace {
// 32 columns by 32 strands of rows; the strands' sums are added in order. The
// first `split` columns go to `out`, the others to `rest`.
__global__ void __launch_bounds__(1024)
sum_rows_kernel(const float* __restrict__ part, int64_t rows, int64_t n, int64_t split,
                float* __restrict__ out, float* __restrict__ rest) {
  __shared__ float sh[32][33];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int64_t i = (int64_t)blockIdx.x * 32 + x;
  float s = 0.f;
  if (i < n) {
#pragma unroll 4
    for (int64_t r = y; r < rows; r += 32) s += part[r * n + i];
  }
  sh[y][x] = s;
  __syncthreads();
  s = warp_sum(sh[x][y]);       // column y of the 32, over the strands
  const int64_t c = (int64_t)blockIdx.x * 32 + y;
  if (x == 0 && c < n) {
    if (c < split)
      out[c] = s;
    else if (rest)
      rest[c - split] = s;
  }
}
}  // namespace

cudaError_t launch_sum_rows(const float* part, int64_t rows, int64_t n, int64_t split, float* out,
                            float* rest, cudaStream_t stream) {
  launch_detail::clear_stale_error();
  sum_rows_kernel<<<(unsigned)ceil_div(n, 32), 1024, 0, stream>>>(part, rows, n, split, out, rest);
  return cudaGetLastError();
}

}  // namespace seq
}  // namespace ferrum
