// Long causal convolution along the last axis of (batch, channels, length):
//   y[t] = sum_{s <= min(t, K-1)} k[s] x[t-s] + skip x[t]
// by its definition: one thread per output. Gradients:
//   dx[t] = sum_{s < K, t+s < L} k[s] dy[t+s] + skip dy[t]
//   dk[s] = sum_b sum_t dy[t] x[t-s],   dskip = sum_b sum_t dy[t] x[t]
#include "seq_common.cuh"

namespace ferrum {
namespace seq {
namespace {

constexpr int kThreads = 256;

struct LongSizes {
  int64_t batch, channels, length, taps, blocks;  // blocks: thread blocks per row
};

template <class T>
__global__ void __launch_bounds__(kThreads)
direct_kernel(Rows<T> x, Rows<T> y, const float* __restrict__ k, const float* __restrict__ skip,
              LongSizes s, bool transposed, int64_t xs, int64_t ys) {
  const int64_t row = blockIdx.x / s.blocks;
  const int64_t t = (blockIdx.x % s.blocks) * kThreads + threadIdx.x;
  if (t >= s.length) return;
  const int64_t b = row / s.channels, d = row % s.channels;
  const T* xr = x.at(b, d);
  const float* kd = k + d * s.taps;
  const int64_t reach = transposed ? s.length - 1 - t : t;
  const int64_t n = reach < s.taps - 1 ? reach : s.taps - 1;
  float v = skip ? skip[d] * to_f(xr[t * xs]) : 0.f;
  for (int64_t i = 0; i <= n; ++i) v = fmaf(kd[i], to_f(xr[(transposed ? t + i : t - i) * xs]), v);
  y.at(b, d)[t * ys] = from_f<T>(v);
}

template <class T>
__global__ void __launch_bounds__(kThreads)
direct_dk_kernel(Rows<T> x, Rows<T> dy, float* __restrict__ dk, float* __restrict__ dskip,
                 LongSizes s, int64_t blocks, int64_t xs, int64_t gs) {
  const int64_t d = blockIdx.x / blocks;
  const int64_t i = (blockIdx.x % blocks) * kThreads + threadIdx.x;
  if (i >= s.taps) return;
  float v = 0.f;
  for (int64_t b = 0; b < s.batch; ++b) {
    float r = 0.f;
    const T *xr = x.at(b, d), *g = dy.at(b, d);
    for (int64_t t = i; t < s.length; ++t) r = fmaf(to_f(g[t * gs]), to_f(xr[(t - i) * xs]), r);
    v += r;
  }
  dk[d * s.taps + i] = v;
  if (dskip && i == 0) dskip[d] = v;
}

// One token: x goes into the history at its sequence's position, and the
// history up to there, reversed, meets the filter. One block per (b, d).
template <class T>
__global__ void __launch_bounds__(kThreads)
long_step_kernel(Rows<T> x, Rows<T> y, Rows<T> hist, const int32_t* __restrict__ positions,
                 const float* __restrict__ k, const float* __restrict__ skip, LongSizes s) {
  __shared__ float sh[kThreads / 32];
  const int64_t b = blockIdx.x / s.channels, d = blockIdx.x % s.channels;
  const int64_t pos = positions[b];
  if (pos < 0 || pos >= s.length) {
    if (threadIdx.x == 0) y.at(b, 0)[d] = from_f<T>(0.f);
    return;
  }
  const T xv = x.at(b, 0)[d];
  T* h = hist.at(b, d);
  const float* kd = k + d * s.taps;
  if (threadIdx.x == 0) h[pos] = xv;
  float v = 0.f;
  for (int64_t i = 1 + threadIdx.x; i <= pos && i < s.taps; i += kThreads)
    v = fmaf(kd[i], to_f(h[pos - i]), v);
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    v = kd[0] * to_f(xv);
    for (int i = 0; i < kThreads / 32; ++i) v += sh[i];
    if (skip) v = fmaf(skip[d], to_f(xv), v);
    y.at(b, 0)[d] = from_f<T>(v);
  }
}

ferrum_status check_long(const ferrum_device* dev, const ferrum_long_conv_args* a, const char* what,
                         bool bwd, bool step) {
  if (ferrum_status s = check_args(dev, a, what)) return s;
  if (a->length > FERRUM_LONG_CONV_MAX_LENGTH)
    return invalid(what, "length must be at most 2^25, got " + std::to_string(a->length));
  const bool none = a->batch == 0 || a->channels == 0, empty = none || a->length == 0;
  if (a->length > 0 && (a->kernel_length < 1 || a->kernel_length > a->length))
    return invalid(what, "kernel_length must be in [1, length], got " +
                             std::to_string(a->kernel_length));
  if (step && !none && a->length == 0) return invalid(what, "the history is empty");
  if (bounded_product({a->batch, a->channels, a->length}) < 0)
    return invalid(what, "batch * channels * length is too large");
  const size_t e = dtype_size(a->dtype);
  if (ferrum_status s = check_ptr(a->kernel, 4, empty, what, "kernel")) return s;
  if (ferrum_status s = check_ptr(a->skip, 4, true, what, "skip")) return s;
  if (ferrum_status s = check_ptr(a->x.ptr, e, empty, what, "x")) return s;
  if (step) {
    if (ferrum_status s = check_ptr(a->history.ptr, e, empty, what, "history")) return s;
    if (ferrum_status s = check_ptr(a->positions, 4, empty, what, "positions")) return s;
  }
  const int64_t out_step = bwd ? a->dx_step : a->y_step;
  if (!step && a->length > 1 && out_step == 0) return invalid(what, "the output's step is 0");
  if (!bwd) return check_ptr(a->y.ptr, e, empty, what, "y");
  if (ferrum_status s = check_ptr(a->dy.ptr, e, empty, what, "dy")) return s;
  if (ferrum_status s = check_ptr(a->dx.ptr, e, empty, what, "dx")) return s;
  if (ferrum_status s = check_ptr(a->dkernel, 4, a->channels == 0 || a->length == 0, what, "dkernel"))
    return s;
  return check_ptr(a->dskip, 4, true, what, "dskip");
}

LongSizes long_sizes(const ferrum_long_conv_args* a) {
  return LongSizes{(int64_t)a->batch, (int64_t)a->channels, (int64_t)a->length,
                   (int64_t)a->kernel_length, ceil_div((int64_t)a->length, kThreads)};
}

}  // namespace
}  // namespace seq
}  // namespace ferrum

using namespace ferrum;
using namespace ferrum::seq;

extern "C" {

ferrum_status ferrum_long_conv(ferrum_device* dev, const ferrum_long_conv_args* a, void* stream) {
  const char* what = "long_conv";
  return guarded(what, [&]() -> ferrum_status {
    if (ferrum_status s = check_long(dev, a, what, false, false)) return s;
    if (a->batch == 0 || a->channels == 0 || a->length == 0) return FERRUM_OK;
    const LongSizes s = long_sizes(a);
    const int64_t blocks = s.batch * s.channels * s.blocks;
    if (blocks > 0x7fffffff) return invalid(what, "too many blocks for one launch");
    DeviceGuard guard(dev->ordinal);
    if (guard.status() != cudaSuccess) return cuda_error(guard.status(), "cudaSetDevice");
    return with_dtype(a->dtype, [&](auto tag) {
      using T = decltype(tag);
      launch_detail::clear_stale_error();
      direct_kernel<T><<<(unsigned)blocks, kThreads, 0, (cudaStream_t)stream>>>(
          rows_of<T>(a->x), rows_of<T>(a->y), a->kernel, a->skip, s, false, a->x_step,
          a->y_step);
      return launched(what);
    });
  });
}

ferrum_status ferrum_long_conv_bwd(ferrum_device* dev, const ferrum_long_conv_args* a,
                                   void* stream) {
  const char* what = "long_conv_bwd";
  return guarded(what, [&]() -> ferrum_status {
    if (ferrum_status s = check_long(dev, a, what, true, false)) return s;
    if (a->channels == 0 || a->length == 0) return FERRUM_OK;
    const LongSizes s = long_sizes(a);
    const int64_t blocks = s.batch * s.channels * s.blocks;
    const int64_t kb = ceil_div(s.taps, kThreads);
    if (blocks > 0x7fffffff || kb * s.channels > 0x7fffffff)
      return invalid(what, "too many blocks for one launch");
    DeviceGuard guard(dev->ordinal);
    if (guard.status() != cudaSuccess) return cuda_error(guard.status(), "cudaSetDevice");
    return with_dtype(a->dtype, [&](auto tag) {
      using T = decltype(tag);
      launch_detail::clear_stale_error();
      if (blocks > 0)
        direct_kernel<T><<<(unsigned)blocks, kThreads, 0, (cudaStream_t)stream>>>(
            rows_of<T>(a->dy), rows_of<T>(a->dx), a->kernel, a->skip, s, true, a->dy_step,
            a->dx_step);
      direct_dk_kernel<T><<<(unsigned)(kb * s.channels), kThreads, 0, (cudaStream_t)stream>>>(
          rows_of<T>(a->x), rows_of<T>(a->dy), a->dkernel, a->dskip, s, kb, a->x_step,
          a->dy_step);
      return launched(what);
    });
  });
}

ferrum_status ferrum_long_conv_step(ferrum_device* dev, const ferrum_long_conv_args* a,
                                    void* stream) {
  const char* what = "long_conv_step";
  return guarded(what, [&]() -> ferrum_status {
    if (ferrum_status s = check_long(dev, a, what, false, true)) return s;
    if (a->batch == 0 || a->channels == 0) return FERRUM_OK;
    const LongSizes s = long_sizes(a);
    if (s.batch * s.channels > 0x7fffffff) return invalid(what, "too many blocks for one launch");
    DeviceGuard guard(dev->ordinal);
    if (guard.status() != cudaSuccess) return cuda_error(guard.status(), "cudaSetDevice");
    return with_dtype(a->dtype, [&](auto tag) {
      using T = decltype(tag);
      launch_detail::clear_stale_error();
      long_step_kernel<T><<<(unsigned)(s.batch * s.channels), kThreads, 0, (cudaStream_t)stream>>>(
          rows_of<T>(a->x), rows_of<T>(a->y), rows_of<T>(a->history), a->positions, a->kernel,
          a->skip, s);
      return launched(what);
    });
  });
}

}  // extern "C"
