// Short causal depthwise convolution over (batch, length, channels):
//   p[t] = bias + sum_j w[j] x[t-K+1+j],  y = p or p * sigmoid(p)
// One thread owns one channel over a run of steps and slides a window of K
// values through registers, so x is read once (and K-1 values again at the
// start of each run); lanes span adjacent channels, so rows are read in whole
// segments. The work is 2K operations per 2 moved values: bound by HBM.
//
// Gradient, with g[t] = dy[t] * act'(p[t]):
//   dx[s] = sum_j w[j] g[s+K-1-j],  dw[j] = sum_t g[t] x[t-K+1+j],  db = sum_t g[t]
// The same run of steps recomputes p; the per-run sums of dw and db go to a
// workspace and are added in a fixed order.
#include "seq_common.cuh"

namespace ferrum {
namespace seq {
namespace {

constexpr int kThreads = 256;
constexpr int kRun = 64;  // steps per thread

struct ConvSizes {
  int64_t batch, length, channels, runs, col_blocks;
};

__device__ __forceinline__ int64_t valid_length(const int32_t* lengths, int64_t b, int64_t length) {
  if (lengths == nullptr) return length;
  const int64_t n = lengths[b];
  return n < 0 ? 0 : (n > length ? length : n);
}

// x at step t (t >= -(K-1)) of one channel: the state in front of the
// sequence, zero past its end.
template <class T, int K>
__device__ __forceinline__ float conv_in(const Rows<T>& x, const T* st, int64_t b, int64_t t,
                                         int64_t d, int64_t len, int64_t channels) {
  if (t >= 0) return t < len ? to_f(x.at(b, t)[d]) : 0.f;
  return st ? to_f(st[(b * (K - 1) + (t + K - 1)) * channels + d]) : 0.f;
}

template <class T, int K>
__global__ void __launch_bounds__(kThreads)
conv1d_fwd_kernel(Rows<T> x, Rows<T> y, const float* __restrict__ weight,
                  const float* __restrict__ bias, const T* st, T* fin,
                  const int32_t* __restrict__ lengths, ConvSizes s, bool silu) {
  int64_t q = blockIdx.x;
  const int64_t d = (q % s.col_blocks) * kThreads + threadIdx.x;
  q /= s.col_blocks;
  const int64_t t0 = (q % s.runs) * kRun, b = q / s.runs;
  if (d >= s.channels) return;
  const int64_t len = valid_length(lengths, b, s.length);
  float w[K], win[K];
#pragma unroll
  for (int j = 0; j < K; ++j) w[j] = weight[d * K + j];
  const float bs = bias ? bias[d] : 0.f;
#pragma unroll
  for (int j = 1; j < K; ++j) win[j] = conv_in<T, K>(x, st, b, t0 - K + j, d, len, s.channels);
  const int64_t t1 = t0 + kRun < s.length ? t0 + kRun : s.length;
  for (int64_t t = t0; t < t1; ++t) {
#pragma unroll
    for (int j = 0; j + 1 < K; ++j) win[j] = win[j + 1];
    win[K - 1] = t < len ? to_f(x.at(b, t)[d]) : 0.f;
    float p = bs;
#pragma unroll
    for (int j = 0; j < K; ++j) p = fmaf(w[j], win[j], p);
    if (silu) p *= sigmoid_f(p);
    y.at(b, t)[d] = from_f<T>(t < len ? p : 0.f);
  }
  if (t0 == 0 && fin != nullptr) {
    // all reads come first: fin may be the initial state's array
    T keep[K];
#pragma unroll
    for (int i = 0; i + 1 < K; ++i)
      keep[i] = from_f<T>(conv_in<T, K>(x, st, b, len - (K - 1) + i, d, len, s.channels));
#pragma unroll
    for (int i = 0; i + 1 < K; ++i) fin[(b * (K - 1) + i) * s.channels + d] = keep[i];
  }
}

template <class T, int K>
__global__ void __launch_bounds__(kThreads)
conv1d_bwd_kernel(Rows<T> x, Rows<T> dy, Rows<T> dx, const float* __restrict__ weight,
                  const float* __restrict__ bias, const T* st, const T* dfin, T* dst,
                  const int32_t* __restrict__ lengths, float* __restrict__ part, ConvSizes s,
                  bool silu) {
  int64_t q = blockIdx.x;
  const int64_t d = (q % s.col_blocks) * kThreads + threadIdx.x;
  q /= s.col_blocks;
  const int64_t run = q % s.runs, t0 = run * kRun, b = q / s.runs;
  if (d >= s.channels) return;
  const int64_t len = valid_length(lengths, b, s.length);
  float w[K], win[K], g[K], dw[K], db = 0.f;
#pragma unroll
  for (int j = 0; j < K; ++j) w[j] = weight[d * K + j], dw[j] = 0.f, g[j] = 0.f;
  const float bs = bias ? bias[d] : 0.f;
#pragma unroll
  for (int j = 1; j < K; ++j) win[j] = conv_in<T, K>(x, st, b, t0 - K + j, d, len, s.channels);
  const int64_t t1 = t0 + kRun < s.length ? t0 + kRun : s.length;
  // g[j] holds the gradient of p at step t-K+1+j; after it moved on to step t,
  // dx of step t-K+1 is complete.
  for (int64_t t = t0; t < t1 + K - 1; ++t) {
#pragma unroll
    for (int j = 0; j + 1 < K; ++j) win[j] = win[j + 1], g[j] = g[j + 1];
    float gt = 0.f;
    win[K - 1] = 0.f;
    if (t < len) {
      win[K - 1] = to_f(x.at(b, t)[d]);
      gt = to_f(dy.at(b, t)[d]);
      if (silu) {
        float p = bs;
#pragma unroll
        for (int j = 0; j < K; ++j) p = fmaf(w[j], win[j], p);
        const float sg = sigmoid_f(p);
        gt *= sg * (1.f + p * (1.f - sg));
      }
      if (t < t1) {
        db += gt;
#pragma unroll
        for (int j = 0; j < K; ++j) dw[j] = fmaf(gt, win[j], dw[j]);
      }
    }
    g[K - 1] = gt;
    const int64_t r = t - K + 1;
    if (r < t0 && !(t0 == 0 && dst != nullptr)) continue;
    float o = 0.f;
#pragma unroll
    for (int j = 0; j < K; ++j) o = fmaf(w[j], g[K - 1 - j], o);
    // a final state is the input's last K-1 values
    const int64_t i = r - (len - (K - 1));
    if (dfin != nullptr && i >= 0 && i < K - 1)
      o += to_f(dfin[(b * (K - 1) + i) * s.channels + d]);
    if (r >= 0)
      dx.at(b, r)[d] = from_f<T>(r < len ? o : 0.f);
    else if (r >= -(K - 1))
      dst[(b * (K - 1) + (r + K - 1)) * s.channels + d] = from_f<T>(o);
  }
  float* o = part + (b * s.runs + run) * (K + 1) * s.channels;
#pragma unroll
  for (int j = 0; j < K; ++j) o[d * K + j] = dw[j];
  o[K * s.channels + d] = db;
}

template <class F>
ferrum_status with_taps(int taps, F f) {
  switch (taps) {
    case 1: return f(std::integral_constant<int, 1>());
    case 2: return f(std::integral_constant<int, 2>());
    case 3: return f(std::integral_constant<int, 3>());
    case 4: return f(std::integral_constant<int, 4>());
    case 5: return f(std::integral_constant<int, 5>());
    case 6: return f(std::integral_constant<int, 6>());
    case 7: return f(std::integral_constant<int, 7>());
    default: return f(std::integral_constant<int, 8>());
  }
}

ferrum_status check_conv(const ferrum_device* dev, const ferrum_conv1d_args* a, const char* what,
                         bool bwd) {
  if (ferrum_status s = check_args(dev, a, what)) return s;
  if (a->taps < 1 || a->taps > FERRUM_CONV1D_MAX_TAPS)
    return invalid(what, "taps must be in [1, 8], got " + std::to_string(a->taps));
  if (bounded_product({a->batch, a->length + (size_t)a->taps, a->channels}) < 0)
    return invalid(what, "batch * length * channels is too large");
  const size_t e = dtype_size(a->dtype);
  const bool none = a->batch == 0 || a->channels == 0, empty = none || a->length == 0;
  if (ferrum_status s = check_ptr(a->weight, 4, none, what, "weight")) return s;
  if (ferrum_status s = check_ptr(a->bias, 4, true, what, "bias")) return s;
  if (ferrum_status s = check_ptr(a->initial_state, e, true, what, "initial_state")) return s;
  if (ferrum_status s = check_ptr(a->lengths, 4, true, what, "lengths")) return s;
  if (ferrum_status s = check_ptr(a->x.ptr, e, empty, what, "x")) return s;
  if (!bwd) {
    if (ferrum_status s = check_ptr(a->y.ptr, e, empty, what, "y")) return s;
    return check_ptr(a->final_state, e, true, what, "final_state");
  }
  if (ferrum_status s = check_ptr(a->dy.ptr, e, empty, what, "dy")) return s;
  if (ferrum_status s = check_ptr(a->dx.ptr, e, empty, what, "dx")) return s;
  if (ferrum_status s = check_ptr(a->dfinal_state, e, true, what, "dfinal_state")) return s;
  if (ferrum_status s = check_ptr(a->dinitial_state, e, true, what, "dinitial_state")) return s;
  if (ferrum_status s = check_ptr(a->dweight, 4, a->channels == 0, what, "dweight")) return s;
  return check_ptr(a->dbias, 4, true, what, "dbias");
}

ConvSizes conv_sizes(const ferrum_conv1d_args* a) {
  ConvSizes s;
  s.batch = (int64_t)a->batch, s.length = (int64_t)a->length, s.channels = (int64_t)a->channels;
  s.runs = s.length > 0 ? ceil_div(s.length, kRun) : 1;  // an empty prompt still copies its state
  s.col_blocks = ceil_div(s.channels, kThreads);
  return s;
}

ferrum_status grid_ok(int64_t blocks, const char* what) {
  return blocks > 0x7fffffff ? invalid(what, "too many blocks for one launch") : FERRUM_OK;
}

ferrum_status conv_fwd(ferrum_device* dev, const ferrum_conv1d_args* a, cudaStream_t stream,
                       const char* what) {
  if (a->batch == 0 || a->channels == 0) return FERRUM_OK;
  const ConvSizes s = conv_sizes(a);
  const int64_t blocks = s.batch * s.runs * s.col_blocks;
  if (ferrum_status st = grid_ok(blocks, what)) return st;
  DeviceGuard guard(dev->ordinal);
  if (guard.status() != cudaSuccess) return cuda_error(guard.status(), "cudaSetDevice");
  return with_dtype(a->dtype, [&](auto tag) {
    using T = decltype(tag);
    return with_taps(a->taps, [&](auto k) {
      launch_detail::clear_stale_error();
      conv1d_fwd_kernel<T, decltype(k)::value><<<(unsigned)blocks, kThreads, 0, stream>>>(
          rows_of<T>(a->x), rows_of<T>(a->y), a->weight, a->bias, (const T*)a->initial_state,
          (T*)a->final_state, a->lengths, s, a->silu != 0);
      return launched(what);
    });
  });
}

}  // namespace
}  // namespace seq
}  // namespace ferrum

using namespace ferrum;
using namespace ferrum::seq;

extern "C" {

ferrum_status ferrum_causal_conv1d(ferrum_device* dev, const ferrum_conv1d_args* a, void* stream) {
  const char* what = "causal_conv1d";
  return guarded(what, [&]() -> ferrum_status {
    if (ferrum_status s = check_conv(dev, a, what, false)) return s;
    return conv_fwd(dev, a, (cudaStream_t)stream, what);
  });
}

ferrum_status ferrum_causal_conv1d_step(ferrum_device* dev, const ferrum_conv1d_args* a,
                                        void* stream) {
  const char* what = "causal_conv1d_step";
  return guarded(what, [&]() -> ferrum_status {
    if (ferrum_status s = check_conv(dev, a, what, false)) return s;
    if (a->length != 1) return invalid(what, "length must be 1, got " + std::to_string(a->length));
    if (a->taps > 1 && a->batch > 0 && a->channels > 0 &&
        (a->initial_state == nullptr || a->final_state == nullptr))
      return invalid(what, "initial_state and final_state are required");
    return conv_fwd(dev, a, (cudaStream_t)stream, what);
  });
}

ferrum_status ferrum_causal_conv1d_bwd(ferrum_device* dev, const ferrum_conv1d_args* a,
                                       void* stream) {
  const char* what = "causal_conv1d_bwd";
  return guarded(what, [&]() -> ferrum_status {
    if (ferrum_status s = check_conv(dev, a, what, true)) return s;
    if (a->channels == 0) return FERRUM_OK;
    cudaStream_t st = (cudaStream_t)stream;
    const ConvSizes z = conv_sizes(a);
    const int64_t parts = z.batch * z.runs, blocks = parts * z.col_blocks;
    if (ferrum_status s = grid_ok(blocks, what)) return s;
    DeviceGuard guard(dev->ordinal);
    if (guard.status() != cudaSuccess) return cuda_error(guard.status(), "cudaSetDevice");
    const int64_t cols = (int64_t)(a->taps + 1) * z.channels;
    PoolBuffer ws(dev, (size_t)(parts * cols) * 4 + 4, st);
    PoolBuffer sums(dev, (size_t)cols * 4, st);
    if (ws.status() != cudaSuccess) return cuda_error(ws.status(), "workspace");
    if (sums.status() != cudaSuccess) return cuda_error(sums.status(), "workspace");
    if (parts > 0) {
      ferrum_status s = with_dtype(a->dtype, [&](auto tag) {
        using T = decltype(tag);
        return with_taps(a->taps, [&](auto k) {
          launch_detail::clear_stale_error();
          conv1d_bwd_kernel<T, decltype(k)::value><<<(unsigned)blocks, kThreads, 0, st>>>(
              rows_of<T>(a->x), rows_of<T>(a->dy), rows_of<T>(a->dx), a->weight, a->bias,
              (const T*)a->initial_state, (const T*)a->dfinal_state, (T*)a->dinitial_state,
              a->lengths, ws.as<float>(), z, a->silu != 0);
          return launched(what);
        });
      });
      if (s) return s;
    }
    cudaError_t e = launch_sum_rows(ws.as<float>(), parts, cols, sums.as<float>(), st);
    if (e != cudaSuccess) return cuda_error(e, what);
    e = cudaMemcpyAsync(a->dweight, sums.as<float>(), (size_t)a->taps * z.channels * 4,
                        cudaMemcpyDeviceToDevice, st);
    if (e == cudaSuccess && a->dbias)
      e = cudaMemcpyAsync(a->dbias, sums.as<float>() + a->taps * z.channels,
                          (size_t)z.channels * 4, cudaMemcpyDeviceToDevice, st);
    return e == cudaSuccess ? FERRUM_OK : cuda_error(e, what);
  });
}

}  // extern "C"
