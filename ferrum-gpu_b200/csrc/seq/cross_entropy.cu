// Softmax cross entropy of hidden rows against a vocabulary matrix: C entries.
#include "cross_entropy.cuh"

namespace ferrum {
namespace seq {
namespace {

// A row's loss from its tiles' statistics: 32 rows by 32 strands of tiles a block,
// joined in a fixed order.
__global__ void __launch_bounds__(1024)
finish_loss_kernel(const RowStat* __restrict__ stats, int tiles, int64_t tokens, int64_t vocab,
                   const int64_t* __restrict__ targets, const float* __restrict__ at_target,
                   float* __restrict__ loss, float* __restrict__ lse) {
  __shared__ RowStat part[32][33];
  await_previous();
  const int x = threadIdx.x % 32, y = threadIdx.x / 32;
  const int64_t t = (int64_t)blockIdx.x * 32 + x;
  RowStat s = {-INFINITY, 0.f};
  if (t < tokens) {
#pragma unroll 4
    for (int i = y; i < tiles; i += 32) s = join(s, stats[(int64_t)i * tokens + t]);
  }
  part[y][x] = s;
  __syncthreads();
  s = part[x][y];                     // row y, strand x
#pragma unroll
  for (int o = 16; o > 0; o /= 2) {
    RowStat q;
    q.top = __shfl_down_sync(0xffffffffu, s.top, o), q.sum = __shfl_down_sync(0xffffffffu, s.sum, o);
    s = join(s, q);
  }
  const int64_t r = (int64_t)blockIdx.x * 32 + y;
  if (x != 0 || r >= tokens) return;
  const bool counts = has_loss(targets[r], vocab);
  const float v = lse_of(s);
  lse[r] = counts ? v : 0.f;
  loss[r] = counts ? v - at_target[r] : 0.f;
}

ferrum_status check_loss(const ferrum_device* dev, const ferrum_cross_entropy_args* a,
                         const char* what, bool bwd) {
  if (ferrum_status s = check_args(dev, a, what)) return s;
  if (a->width < 1) return invalid(what, "width must be at least 1");
  if (a->vocab < 1) return invalid(what, "vocab must be at least 1");
  // (rows are numbered by 32 bits in the tensor copies)
  if (a->tokens > 0x7fffff00 || a->vocab > 0x7fffff00 || a->width > 0x7fffff00)
    return invalid(what, "tokens, vocab and width must be below 2^31 - 256");
  // The tensor cores cut off each of the width / 16 additions of a logit in the gradient, which
  // shrinks it by 1.5e-8 of it each: at 2^16 that is 6e-5 of the logit, and the softmax of one of
  // 2.5 off by a third of float16's rounding, in one direction. (At 2^26 a tile also takes 0.3 of
  // the second that waits are given.)
  if (bwd && a->dtype != FERRUM_F32 && a->width > FERRUM_LOSS_BWD_MAX_WIDTH_16)
    return invalid(what, "width must be at most 2^16 in 16-bit types");
  if (bounded_product({a->tokens, a->width}) < 0 || bounded_product({a->vocab, a->width}) < 0)
    return invalid(what, "tokens * width or vocab * width is too large");
  const size_t e = dtype_size(a->dtype);
  const bool none = a->tokens == 0;
  struct {
    const void* p;
    size_t align;
    bool optional;
    const char* name;
  } const arrays[] = {
      {a->x, e, none, "x"},
      {a->weight, e, false, "weight"},
      {a->targets, 8, none, "targets"},
      {a->loss, 4, bwd || none, "loss"},
      {a->lse, 4, none, "lse"},
      {a->dloss, 4, true, "dloss"},
      {a->dlse, 4, true, "dlse"},
      {a->dx, e, !bwd || none, "dx"},
      {a->dweight, e, !bwd, "dweight"},
  };
  for (const auto& v : arrays)
    if (ferrum_status s = check_ptr(v.p, v.align, v.optional, what, v.name)) return s;
  return FERRUM_OK;
}

}  // namespace

ferrum_status finish_loss(const RowStat* stats, int parts, const float* at_target,
                          const ferrum_cross_entropy_args* a, cudaStream_t stream, const char* what) {
  const int64_t n = (int64_t)a->tokens;
  return start(what, false, finish_loss_kernel, ceil_div(n, 32), 1024, 0, stream, stats, parts, n,
               (int64_t)a->vocab, a->targets, at_target, a->loss, a->lse);
}

}  // namespace seq
}  // namespace ferrum

using namespace ferrum;
using namespace ferrum::seq;

extern "C" {

ferrum_status ferrum_linear_cross_entropy(ferrum_device* dev, const ferrum_cross_entropy_args* a,
                                          void* stream) {
  const char* what = "linear_cross_entropy";
  return guarded(what, [&]() -> ferrum_status {
    if (ferrum_status s = check_loss(dev, a, what, false)) return s;
    if (a->tokens == 0) return FERRUM_OK;
    DeviceGuard guard(dev->ordinal);
    if (guard.status() != cudaSuccess) return cuda_error(guard.status(), "cudaSetDevice");
    launch_detail::clear_stale_error();
    return a->dtype == FERRUM_F32 ? loss_fwd_f32(dev, a, (cudaStream_t)stream, what)
                                  : loss_fwd_tc(dev, a, (cudaStream_t)stream, what);
  });
}

ferrum_status ferrum_linear_cross_entropy_bwd(ferrum_device* dev,
                                              const ferrum_cross_entropy_args* a, void* stream) {
  const char* what = "linear_cross_entropy_bwd";
  return guarded(what, [&]() -> ferrum_status {
    if (ferrum_status s = check_loss(dev, a, what, true)) return s;
    DeviceGuard guard(dev->ordinal);
    if (guard.status() != cudaSuccess) return cuda_error(guard.status(), "cudaSetDevice");
    cudaStream_t st = (cudaStream_t)stream;
    if (a->tokens == 0) {      // no gradient of the weights
      cudaError_t e = cudaMemset2DAsync(a->dweight, (size_t)a->dweight_stride * dtype_size(a->dtype), 0,
                                        a->width * dtype_size(a->dtype), a->vocab, st);
      return e == cudaSuccess ? FERRUM_OK : cuda_error(e, what);
    }
    launch_detail::clear_stale_error();
    return a->dtype == FERRUM_F32 ? loss_bwd_f32(dev, a, st, what) : loss_bwd_tc(dev, a, st, what);
  });
}

}  // extern "C"
