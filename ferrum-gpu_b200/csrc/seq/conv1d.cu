// Short causal depthwise convolution over (batch, length, channels):
//   p[t] = bias + sum_j w[j] x[t-K+1+j],  y = p or p * sigmoid(p)
// The work is 2K operations per 2 moved values: bound by HBM. A thread owns
// two adjacent channels (one where the rows are not aligned) over a run of
// steps and slides a window of K values through registers, so x is read once,
// and K-1 rows again at the start of each run. It loads 8 rows ahead of using
// them (4 in the gradient). Bytes in flight decide: 8 x 2048 x 4096, 4 taps,
// bf16 took 75 us with 4 channels, 4 rows ahead and 24 warps an SM, 92 with 8
// channels and 16 warps, 70 with 2 channels, 8 rows and 32 warps; the
// gradient 142 with 24 warps and 131 with 32 (float32, whose windows spill
// there, 162 and 181; forward 95). That is 3.9 and 3.1 TB/s of the 6.5 of a copy, bound by
// issue slots (61 and 72 %) and, forward, the SiLU's two special functions a
// value (53 %). Runs are long (64 steps) where the batch fills the GPU
// and shorter where it does not.
//
// Gradient, with g[t] = dy[t] * act'(p[t]):
//   dx[s] = sum_j w[j] g[s+K-1-j],  dw[j] = sum_t g[t] x[t-K+1+j],  db = sum_t g[t]
// The same run of steps recomputes p; the per-run sums of dw and db go to a
// workspace and are added in a fixed order.
#include <algorithm>
#include <type_traits>

#include "seq_common.cuh"

namespace ferrum {
namespace seq {
namespace {

constexpr int kThreads = 128;
constexpr int kAhead = 8, kAheadBwd = 4;   // rows loaded ahead

struct ConvSizes {
  int64_t batch, length, channels, run, runs, col_blocks;
};

__device__ __forceinline__ int64_t valid_length(const int32_t* lengths, int64_t b, int64_t length) {
  if (lengths == nullptr) return length;
  const int64_t n = lengths[b];
  return n < 0 ? 0 : (n > length ? length : n);
}

template <int VL>
__device__ __forceinline__ void clear(float (&v)[VL]) {
#pragma unroll
  for (int e = 0; e < VL; ++e) v[e] = 0.f;
}

// x at step t (t >= -(K-1)) of VL channels: the state in front of the
// sequence, zero past its end.
template <class T, int K, int VL>
__device__ __forceinline__ void conv_in(const Rows<T>& x, const T* st, int64_t b, int64_t t,
                                        int64_t d, int64_t len, int64_t channels, float (&v)[VL]) {
  clear(v);
  if (t >= 0) {
    if (t < len) load_vec<T, VL>(x.at(b, t) + d, v);
  } else if (st) {
    load_vec<T, VL>(st + (b * (K - 1) + (t + K - 1)) * channels + d, v);
  }
}

// Blocks run over (column block, run, sequence).
struct ConvPlace {
  int64_t d, run, b;
  template <int VL>
  static __device__ __forceinline__ ConvPlace of(const ConvSizes& s) {
    int64_t q = blockIdx.x;
    ConvPlace p;
    p.d = (q % s.col_blocks * kThreads + threadIdx.x) * VL;
    q /= s.col_blocks;
    p.run = q % s.runs, p.b = q / s.runs;
    return p;
  }
};

template <class T, int K, int VL>
__global__ void __launch_bounds__(kThreads, VL == 1 ? 1 : 8)
conv1d_fwd_kernel(Rows<T> x, Rows<T> y, const float* __restrict__ weight,
                  const float* __restrict__ bias, const T* st, T* fin,
                  const int32_t* __restrict__ lengths, ConvSizes s, bool silu) {
  const ConvPlace at = ConvPlace::of<VL>(s);
  const int64_t d = at.d, b = at.b, t0 = at.run * s.run;
  if (d >= s.channels) return;
  const int64_t len = valid_length(lengths, b, s.length);
  float w[K][VL], win[K][VL], bs[VL];
#pragma unroll
  for (int j = 0; j < K; ++j)
#pragma unroll
    for (int e = 0; e < VL; ++e) w[j][e] = weight[(d + e) * K + j];
#pragma unroll
  for (int e = 0; e < VL; ++e) bs[e] = bias ? bias[d + e] : 0.f;
#pragma unroll
  for (int j = 1; j < K; ++j) conv_in<T, K, VL>(x, st, b, t0 - K + j, d, len, s.channels, win[j]);
  // The run's steps and those of them inside the sequence, from t0 on.
  const int n = (int)(s.length - t0 < s.run ? s.length - t0 : s.run);
  const int valid = len - t0 < n ? (len - t0 < 0 ? 0 : (int)(len - t0)) : n;
  const T* px = x.at(b, t0) + d;
  T* py = y.at(b, t0) + d;
  // kAhead steps from t on; EDGE where some lie past the run or the sequence
  auto block = [&](auto edge, int t) {
    constexpr bool EDGE = decltype(edge)::value;
    float in[kAhead][VL];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (EDGE) clear(in[i]);
      if (!EDGE || t + i < valid) load_vec<T, VL>(px + i * x.st, in[i]);
    }
    px += kAhead * x.st;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (EDGE && t + i >= n) return;
      float p[VL];
#pragma unroll
      for (int e = 0; e < VL; ++e) {
#pragma unroll
        for (int j = 0; j + 1 < K; ++j) win[j][e] = win[j + 1][e];
        win[K - 1][e] = in[i][e];
        float v = bs[e];
#pragma unroll
        for (int j = 0; j < K; ++j) v = fmaf(w[j][e], win[j][e], v);
        if (silu) v *= sigmoid_f(v);
        p[e] = !EDGE || t + i < valid ? v : 0.f;
      }
      store_vec<T, VL>(py, p);
      py += y.st;
    }
  };
  int t = 0;
  for (; t + kAhead <= valid; t += kAhead) block(std::false_type(), t);
  for (; t < n; t += kAhead) block(std::true_type(), t);
  if (t0 == 0 && fin != nullptr) {
    // all reads come first: fin may be the initial state's array
    float keep[K][VL];
#pragma unroll
    for (int i = 0; i + 1 < K; ++i)
      conv_in<T, K, VL>(x, st, b, len - (K - 1) + i, d, len, s.channels, keep[i]);
#pragma unroll
    for (int i = 0; i + 1 < K; ++i)
      store_vec<T, VL>(fin + (b * (K - 1) + i) * s.channels + d, keep[i]);
  }
}

template <class T, int K, int VL>
__global__ void __launch_bounds__(kThreads, VL == 1 ? 1 : (sizeof(T) == 2 ? 8 : 6))
conv1d_bwd_kernel(Rows<T> x, Rows<T> dy, Rows<T> dx, const float* __restrict__ weight,
                  const float* __restrict__ bias, const T* st, const T* dfin, T* dst,
                  const int32_t* __restrict__ lengths, float* __restrict__ part, ConvSizes s,
                  bool silu) {
  const ConvPlace at = ConvPlace::of<VL>(s);
  const int64_t d = at.d, b = at.b, t0 = at.run * s.run;
  if (d >= s.channels) return;
  const int64_t len = valid_length(lengths, b, s.length);
  float w[K][VL], win[K][VL], g[K][VL], dw[K][VL], db[VL], bs[VL];
#pragma unroll
  for (int e = 0; e < VL; ++e) {
    bs[e] = bias ? bias[d + e] : 0.f, db[e] = 0.f;
#pragma unroll
    for (int j = 0; j < K; ++j) w[j][e] = weight[(d + e) * K + j], dw[j][e] = 0.f, g[j][e] = 0.f;
  }
#pragma unroll
  for (int j = 1; j < K; ++j) conv_in<T, K, VL>(x, st, b, t0 - K + j, d, len, s.channels, win[j]);
  // The run's steps and those of them inside the sequence, from t0 on; the
  // gradients of the last K-1 need as many steps of the next run.
  const int n = (int)(s.length - t0 < s.run ? s.length - t0 : s.run);
  const int64_t left = len - t0 < 0 ? 0 : len - t0;
  const int valid = (int)(left < n + K - 1 ? left : n + K - 1);
  const T *px = x.at(b, t0) + d, *pg = dy.at(b, t0) + d;
  T* po = dx.at(b, t0) + d - (K - 1) * dx.st;    // row t-K+1
  // g[j] holds the gradient of p at step t-K+1+j; after it moved on to step t,
  // dx of step t-K+1 is complete. EDGE where steps lie past the run or the
  // sequence, or dx in front of the run, or a final state's gradient joins.
  auto block = [&](auto edge, int t) {
    constexpr bool EDGE = decltype(edge)::value;
    float in[kAheadBwd][VL], gin[kAheadBwd][VL];
#pragma unroll
    for (int i = 0; i < kAheadBwd; ++i) {
      if (EDGE) clear(in[i]), clear(gin[i]);
      if (!EDGE || t + i < valid) {
        load_vec<T, VL>(px + i * x.st, in[i]);
        load_vec<T, VL>(pg + i * dy.st, gin[i]);
      }
    }
    px += kAheadBwd * x.st, pg += kAheadBwd * dy.st;
#pragma unroll
    for (int i = 0; i < kAheadBwd; ++i) {
      if (EDGE && t + i >= n + K - 1) return;
      float o[VL];
#pragma unroll
      for (int e = 0; e < VL; ++e) {
#pragma unroll
        for (int j = 0; j + 1 < K; ++j) win[j][e] = win[j + 1][e], g[j][e] = g[j + 1][e];
        win[K - 1][e] = in[i][e];
        float gt = gin[i][e];
        if (silu) {
          float p = bs[e];
#pragma unroll
          for (int j = 0; j < K; ++j) p = fmaf(w[j][e], win[j][e], p);
          const float sg = sigmoid_f(p);
          gt *= sg * fmaf(p, 1.f - sg, 1.f);
        }
        if (EDGE && t + i >= valid) gt = 0.f;     // whatever the padding's p
        g[K - 1][e] = gt;
        if (!EDGE || t + i < n) {
          db[e] += gt;
#pragma unroll
          for (int j = 0; j < K; ++j) dw[j][e] = fmaf(gt, win[j][e], dw[j][e]);
        }
        o[e] = 0.f;
#pragma unroll
        for (int j = 0; j < K; ++j) o[e] = fmaf(w[j][e], g[K - 1 - j][e], o[e]);
      }
      if constexpr (EDGE) {
        const int64_t r = t0 + t + i - K + 1;
        if (r >= t0 || (t0 == 0 && dst != nullptr)) {
          // a final state is the input's last K-1 values
          const int64_t f = r - (len - (K - 1));
          if (dfin != nullptr && f >= 0 && f < K - 1) {
            float q[VL];
            load_vec<T, VL>(dfin + (b * (K - 1) + f) * s.channels + d, q);
#pragma unroll
            for (int e = 0; e < VL; ++e) o[e] += q[e];
          }
          if (r >= 0) {
            if (r >= len) clear(o);
            store_vec<T, VL>(po, o);
          } else {
            store_vec<T, VL>(dst + (b * (K - 1) + (r + K - 1)) * s.channels + d, o);
          }
        }
      } else {
        store_vec<T, VL>(po, o);
      }
      po += dx.st;
    }
  };
  // steps whose blocks are whole: inside the run and, where a final state has
  // a gradient, in front of its rows
  const int64_t whole64 = dfin != nullptr ? left - (K - 1) : left;
  const int whole = (int)(whole64 < n ? whole64 : n);
  int t = 0;
  for (; t < n + K - 1 && t < K - 1; t += kAheadBwd) block(std::true_type(), t);
  for (; t + kAheadBwd <= whole; t += kAheadBwd) block(std::false_type(), t);
  for (; t < n + K - 1; t += kAheadBwd) block(std::true_type(), t);
  float* o = part + (b * s.runs + at.run) * (K + 1) * s.channels;
#pragma unroll
  for (int e = 0; e < VL; ++e) {
#pragma unroll
    for (int j = 0; j < K; ++j) o[(d + e) * K + j] = dw[j][e];
    o[K * s.channels + d + e] = db[e];
  }
}

// One step of every sequence: K - 1 rows of state and one of x in, the state
// moved up by one row and y out. Each thread owns VL channels of a sequence
// and reads before it writes, so the state may be updated in place.
template <class T, int K, int VL>
__global__ void __launch_bounds__(kThreads)
conv1d_step_kernel(Rows<T> x, Rows<T> y, const float* __restrict__ weight,
                   const float* __restrict__ bias, const T* st, T* fin, int64_t batch,
                   int64_t channels, bool silu) {
  const int64_t per = channels / VL, i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= batch * per) return;
  const int64_t b = i / per, d = i % per * VL;
  float win[K][VL], w[VL * K], p[VL];
#pragma unroll
  for (int j = 0; j + 1 < K; ++j) load_vec<T, VL>(st + (b * (K - 1) + j) * channels + d, win[j]);
  load_vec<T, VL>(x.at(b, 0) + d, win[K - 1]);
  if constexpr (VL % 4 == 0) {       // a channel's taps are adjacent, and 16-byte aligned
    load_vec<float, VL * K>(weight + d * K, w);
  } else {
#pragma unroll
    for (int j = 0; j < VL * K; ++j) w[j] = weight[d * K + j];
  }
#pragma unroll
  for (int e = 0; e < VL; ++e) {
    float v = bias ? bias[d + e] : 0.f;
#pragma unroll
    for (int j = 0; j < K; ++j) v = fmaf(w[e * K + j], win[j][e], v);
    if (silu) v *= sigmoid_f(v);
    p[e] = v;
  }
  store_vec<T, VL>(y.at(b, 0) + d, p);
#pragma unroll
  for (int j = 0; j + 1 < K; ++j) store_vec<T, VL>(fin + (b * (K - 1) + j) * channels + d, win[j + 1]);
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
  if (a->length > (size_t)kMaxElems ||      // (and length + taps would wrap around)
      bounded_product({a->batch, a->length + (size_t)a->taps, a->channels}) < 0)
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

ConvSizes conv_sizes(const ferrum_conv1d_args* a, int vl) {
  ConvSizes s;
  s.batch = (int64_t)a->batch, s.length = (int64_t)a->length, s.channels = (int64_t)a->channels;
  s.col_blocks = ceil_div(s.channels, kThreads * vl);
  // Long runs read few rows twice; short ones give every SM work. 4 blocks an
  // SM, if that takes runs of no less than 8 steps (us, forward and gradient,
  // with runs of 64 and 8 steps: 1 x 1000 x 2048 16.4, 28.9 and 10.2, 22.8;
  // 1 x 8192 x 2048 24.6, 47.4 and 34.8, 82.2).
  s.run = 64;
  while (s.run > 8 && s.batch * s.col_blocks * ceil_div(s.length, s.run) < 148 * 4) s.run /= 2;
  s.runs = s.length > 0 ? ceil_div(s.length, s.run) : 1;  // an empty prompt still copies its state
  return s;
}

ferrum_status grid_ok(int64_t blocks, const char* what) {
  return blocks > 0x7fffffff ? invalid(what, "too many blocks for one launch") : FERRUM_OK;
}

// Whether all arrays can be accessed `bytes` at a time.
bool conv_vec(const ferrum_conv1d_args* a, bool bwd, int vl) {
  const size_t e = dtype_size(a->dtype), bytes = std::min<size_t>(16, vl * e);
  auto ok = [&](const ferrum_rows& r) {
    return aligned(r.ptr, bytes) && r.batch_stride * (int64_t)e % (int64_t)bytes == 0 &&
           r.row_stride * (int64_t)e % (int64_t)bytes == 0;
  };
  bool v = a->channels % vl == 0 && ok(a->x) && aligned(a->initial_state, bytes);
  if (!bwd) return v && ok(a->y) && aligned(a->final_state, bytes);
  return v && ok(a->dy) && ok(a->dx) && aligned(a->dfinal_state, bytes) &&
         aligned(a->dinitial_state, bytes);
}

// f(taps, values per thread): wide accesses for the taps in use (up to 4)
template <int WIDE, class F>
ferrum_status with_conv(int taps, bool vec, F f) {
  return with_taps(taps, [&](auto k) {
    if constexpr (decltype(k)::value <= 4) {
      if (vec) return f(k, std::integral_constant<int, WIDE>());
    }
    return f(k, std::integral_constant<int, 1>());
  });
}

ferrum_status conv_fwd(ferrum_device* dev, const ferrum_conv1d_args* a, cudaStream_t stream,
                       const char* what) {
  if (a->batch == 0 || a->channels == 0) return FERRUM_OK;
  DeviceGuard guard(dev->ordinal);
  if (guard.status() != cudaSuccess) return cuda_error(guard.status(), "cudaSetDevice");
  return with_dtype(a->dtype, [&](auto tag) {
    using T = decltype(tag);
    return with_conv<2>(a->taps, conv_vec(a, false, 2), [&](auto k, auto vl) -> ferrum_status {
      const ConvSizes s = conv_sizes(a, decltype(vl)::value);
      const int64_t blocks = s.batch * s.runs * s.col_blocks;
      if (ferrum_status st = grid_ok(blocks, what)) return st;
      launch_detail::clear_stale_error();
      conv1d_fwd_kernel<T, decltype(k)::value, decltype(vl)::value>
          <<<(unsigned)blocks, kThreads, 0, stream>>>(
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
    if (a->lengths != nullptr) return invalid(what, "lengths does not apply to one step");
    if (a->batch == 0 || a->channels == 0) return FERRUM_OK;
    DeviceGuard guard(dev->ordinal);
    if (guard.status() != cudaSuccess) return cuda_error(guard.status(), "cudaSetDevice");
    return with_dtype(a->dtype, [&](auto tag) {
      using T = decltype(tag);
      const bool vec = conv_vec(a, false, 4) && aligned(a->weight, 16);
      return with_conv<4>(a->taps, vec, [&](auto k, auto vl) -> ferrum_status {
        constexpr int VL = decltype(vl)::value;
        const int64_t blocks = ceil_div((int64_t)a->batch * (int64_t)(a->channels / VL), kThreads);
        if (ferrum_status s = grid_ok(blocks, what)) return s;
        launch_detail::clear_stale_error();
        conv1d_step_kernel<T, decltype(k)::value, VL>
            <<<(unsigned)blocks, kThreads, 0, (cudaStream_t)stream>>>(
                rows_of<T>(a->x), rows_of<T>(a->y), a->weight, a->bias,
                (const T*)a->initial_state, (T*)a->final_state, (int64_t)a->batch,
                (int64_t)a->channels, a->silu != 0);
        return launched(what);
      });
    });
  });
}

ferrum_status ferrum_causal_conv1d_bwd(ferrum_device* dev, const ferrum_conv1d_args* a,
                                       void* stream) {
  const char* what = "causal_conv1d_bwd";
  return guarded(what, [&]() -> ferrum_status {
    if (ferrum_status s = check_conv(dev, a, what, true)) return s;
    if (a->channels == 0) return FERRUM_OK;
    cudaStream_t st = (cudaStream_t)stream;
    DeviceGuard guard(dev->ordinal);
    if (guard.status() != cudaSuccess) return cuda_error(guard.status(), "cudaSetDevice");
    return with_dtype(a->dtype, [&](auto tag) {
      using T = decltype(tag);
      return with_conv<2>(a->taps, conv_vec(a, true, 2), [&](auto k, auto vl) -> ferrum_status {
        const ConvSizes z = conv_sizes(a, decltype(vl)::value);
        const int64_t parts = z.batch * z.runs, blocks = parts * z.col_blocks;
        if (ferrum_status s = grid_ok(blocks, what)) return s;
        const int64_t cols = (int64_t)(a->taps + 1) * z.channels;
        PoolBuffer ws(dev, (size_t)(parts * cols) * 4 + 4, st);
        if (ws.status() != cudaSuccess) return cuda_error(ws.status(), "workspace");
        float* part = ws.as<float>();
        if (parts > 0) {
          launch_detail::clear_stale_error();
          conv1d_bwd_kernel<T, decltype(k)::value, decltype(vl)::value>
              <<<(unsigned)blocks, kThreads, 0, st>>>(
                  rows_of<T>(a->x), rows_of<T>(a->dy), rows_of<T>(a->dx), a->weight, a->bias,
                  (const T*)a->initial_state, (const T*)a->dfinal_state, (T*)a->dinitial_state,
                  a->lengths, part, z, a->silu != 0);
          if (ferrum_status s = launched(what)) return s;
        }
        cudaError_t e =
            launch_sum_rows(part, parts, cols, a->taps * z.channels, a->dweight, a->dbias, st);
        return e == cudaSuccess ? FERRUM_OK : cuda_error(e, what);
      });
    });
  });
}

}  // extern "C"
