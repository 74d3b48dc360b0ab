// Norms around a block, over rows of `channels` values:
//   in front:  r = residual + scale * x,  y = N(r) * weight + bias
//   behind:    p = N(x * silu(gate)) * weight + bias   (gate inside)
//              p = (N(x) * weight + bias) * silu(gate) (gate outside)
//              y = residual + scale * p
// N(v) = (v - m) * i with i = 1 / sqrt(mean((v - m)^2) + eps), m the mean for
// the layer norm and 0 for RMS. With n the normalised values and dn their
// gradient, dv = i * (dn - n * mean(dn * n) - [layer] mean(dn)).
// (A row of one value leaves dn - n * mean(dn * n) = dn (1 - n^2) to a
// difference of equals; there 1 - n^2 = eps i^2 is used instead.)
// A few operations per moved value: bound by HBM. One block per row (behind:
// per group of a row); the parameters' gradients are column sums over the
// rows, taken by a second kernel from the rows' statistics.
#include "seq_common.cuh"

namespace ferrum {
namespace seq {
namespace {

constexpr int kThreads = 256;

// Sum over the block, in every thread, in a fixed order.
__device__ float block_sum(float v, float* sh) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) s += sh[i];
  return s;
}

struct NormArgs {
  int64_t rows, channels, groups, width;  // width = channels / groups
  float eps;
  bool layer, inside;
  const float *weight, *bias, *scale;
  int64_t x_st, gate_st, res_st, y_st, r_st, dy_st, dr_st, dx_st, dgate_st, dres_st;
  float4* stats;  // (rows * groups): mean, 1 / deviation, mean of dn, mean of dn * n
};

// Gradient of a value from that of its normalised value n.
__device__ __forceinline__ float norm_grad(const NormArgs& a, float inv, float dn, float n,
                                           float mean_dn, float mean_dnn) {
  if (a.width == 1) return a.layer ? 0.f : inv * dn * (a.eps * inv * inv);
  return inv * (dn - mean_dn - n * mean_dnn);
}

// r (a row of the residual stream) in front of a block
template <class T, class R>
__device__ __forceinline__ float before_value(const T* x, const R* res, const float* scale,
                                              int64_t c) {
  float v = res ? to_f(res[c]) : 0.f;
  if (x) v = fmaf(scale ? scale[c] : 1.f, to_f(x[c]), v);
  return v;
}

template <class T, class R>
__global__ void __launch_bounds__(kThreads)
norm_before_kernel(NormArgs a, const T* x, const R* res, T* y, R* r) {
  __shared__ float sh[kThreads / 32];
  const int64_t row = blockIdx.x;
  if (x) x += row * a.x_st;
  if (res) res += row * a.res_st;
  y += row * a.y_st;
  float s = 0.f;
  for (int64_t c = threadIdx.x; c < a.channels; c += kThreads)
    s += before_value(x, res, a.scale, c);
  const float mean = a.layer ? block_sum(s, sh) / (float)a.channels : 0.f;
  float q = 0.f;
  for (int64_t c = threadIdx.x; c < a.channels; c += kThreads) {
    const float v = before_value(x, res, a.scale, c) - mean;
    q = fmaf(v, v, q);
  }
  const float inv = 1.f / sqrtf(block_sum(q, sh) / (float)a.channels + a.eps);
  for (int64_t c = threadIdx.x; c < a.channels; c += kThreads) {
    const float v = before_value(x, res, a.scale, c);
    const float n = (v - mean) * inv;
    if (r) r[row * a.r_st + c] = from_f<R>(v);
    y[c] = from_f<T>(fmaf(n, a.weight[c], a.bias ? a.bias[c] : 0.f));
  }
}

template <class T, class R>
__global__ void __launch_bounds__(kThreads)
norm_before_bwd_kernel(NormArgs a, const R* r, const T* dy, const R* dr, T* dx, R* dres) {
  __shared__ float sh[kThreads / 32];
  const int64_t row = blockIdx.x;
  r += row * a.r_st, dy += row * a.dy_st;
  const float w = 1.f / (float)a.channels;
  float s = 0.f;
  for (int64_t c = threadIdx.x; c < a.channels; c += kThreads) s += to_f(r[c]);
  const float mean = a.layer ? block_sum(s, sh) * w : 0.f;
  float q = 0.f, g1 = 0.f, g2 = 0.f;
  for (int64_t c = threadIdx.x; c < a.channels; c += kThreads) {
    const float v = to_f(r[c]) - mean, g = to_f(dy[c]) * a.weight[c];
    q = fmaf(v, v, q), g1 += g, g2 = fmaf(g, v, g2);
  }
  const float inv = 1.f / sqrtf(block_sum(q, sh) * w + a.eps);
  g1 = a.layer ? block_sum(g1, sh) * w : 0.f;
  g2 = block_sum(g2, sh) * w * inv;
  if (threadIdx.x == 0) a.stats[row] = make_float4(mean, inv, g1, g2);
  for (int64_t c = threadIdx.x; c < a.channels; c += kThreads) {
    const float n = (to_f(r[c]) - mean) * inv;
    float o = norm_grad(a, inv, to_f(dy[c]) * a.weight[c], n, g1, g2);
    if (dr) o += to_f(dr[row * a.dr_st + c]);
    if (dres) dres[row * a.dres_st + c] = from_f<R>(o);
    if (dx) dx[row * a.dx_st + c] = from_f<T>(a.scale ? o * a.scale[c] : o);
  }
}

// Column sums over a block's share of the rows: part[(share * 3 + k) * channels + c]
// for k = dweight, dbias, dscale.
template <class T, class R>
__global__ void __launch_bounds__(kThreads)
norm_before_cols_kernel(NormArgs a, const T* x, const R* r, const T* dy, const R* dr,
                        float* part, int64_t col_blocks, int64_t share) {
  const int64_t c = (blockIdx.x % col_blocks) * kThreads + threadIdx.x, p = blockIdx.x / col_blocks;
  if (c >= a.channels) return;
  const int64_t r1 = (p + 1) * share < a.rows ? (p + 1) * share : a.rows;
  const float w = a.weight[c];
  float dw = 0.f, db = 0.f, ds = 0.f;
  for (int64_t i = p * share; i < r1; ++i) {
    const float4 st = a.stats[i];
    const float g = to_f(dy[i * a.dy_st + c]), n = (to_f(r[i * a.r_st + c]) - st.x) * st.y;
    dw = fmaf(g, n, dw);
    db += g;
    if (x) {
      float o = norm_grad(a, st.y, g * w, n, st.z, st.w);
      if (dr) o += to_f(dr[i * a.dr_st + c]);
      ds = fmaf(o, to_f(x[i * a.x_st + c]), ds);
    }
  }
  part[(p * 3 + 0) * a.channels + c] = dw;
  part[(p * 3 + 1) * a.channels + c] = db;
  part[(p * 3 + 2) * a.channels + c] = ds;
}

template <class T>
__device__ __forceinline__ float after_value(const NormArgs& a, const T* x, const T* gate,
                                             int64_t c) {
  float v = to_f(x[c]);
  if (a.inside && gate) {
    const float g = to_f(gate[c]);
    v *= g * sigmoid_f(g);
  }
  return v;
}

template <class T, class R>
__global__ void __launch_bounds__(kThreads)
norm_after_kernel(NormArgs a, const T* x, const T* gate, const R* res, T* y) {
  __shared__ float sh[kThreads / 32];
  const int64_t row = blockIdx.x / a.groups, c0 = (blockIdx.x % a.groups) * a.width,
                c1 = c0 + a.width;
  x += row * a.x_st;
  if (gate) gate += row * a.gate_st;
  if (res) res += row * a.res_st;
  y += row * a.y_st;
  float s = 0.f;
  for (int64_t c = c0 + threadIdx.x; c < c1; c += kThreads) s += after_value(a, x, gate, c);
  const float mean = a.layer ? block_sum(s, sh) / (float)a.width : 0.f;
  float q = 0.f;
  for (int64_t c = c0 + threadIdx.x; c < c1; c += kThreads) {
    const float v = after_value(a, x, gate, c) - mean;
    q = fmaf(v, v, q);
  }
  const float inv = 1.f / sqrtf(block_sum(q, sh) / (float)a.width + a.eps);
  for (int64_t c = c0 + threadIdx.x; c < c1; c += kThreads) {
    float p = fmaf((after_value(a, x, gate, c) - mean) * inv, a.weight[c],
                   a.bias ? a.bias[c] : 0.f);
    if (!a.inside && gate) {
      const float g = to_f(gate[c]);
      p *= g * sigmoid_f(g);
    }
    const float base = res ? to_f(res[c]) : 0.f;
    y[c] = from_f<T>(fmaf(a.scale ? a.scale[c] : 1.f, p, base));
  }
}

// d silu(g) / dg, and silu(g)
__device__ __forceinline__ void silu_grad(float g, float& f, float& df) {
  const float sg = sigmoid_f(g);
  f = g * sg;
  df = sg * (1.f + g * (1.f - sg));
}

template <class T>
__global__ void __launch_bounds__(kThreads)
norm_after_bwd_kernel(NormArgs a, const T* x, const T* gate, const T* dy, T* dx, T* dgate) {
  __shared__ float sh[kThreads / 32];
  const int64_t row = blockIdx.x / a.groups, c0 = (blockIdx.x % a.groups) * a.width,
                c1 = c0 + a.width;
  x += row * a.x_st, dy += row * a.dy_st, dx += row * a.dx_st;
  if (gate) gate += row * a.gate_st, dgate += row * a.dgate_st;
  const float w = 1.f / (float)a.width;
  float s = 0.f;
  for (int64_t c = c0 + threadIdx.x; c < c1; c += kThreads) s += after_value(a, x, gate, c);
  const float mean = a.layer ? block_sum(s, sh) * w : 0.f;
  // gradient of the normalised value of column c
  auto dnorm = [&](int64_t c) {
    float g = to_f(dy[c]) * (a.scale ? a.scale[c] : 1.f) * a.weight[c];
    if (!a.inside && gate) {
      const float z = to_f(gate[c]);
      g *= z * sigmoid_f(z);
    }
    return g;
  };
  float q = 0.f, g1 = 0.f, g2 = 0.f;
  for (int64_t c = c0 + threadIdx.x; c < c1; c += kThreads) {
    const float v = after_value(a, x, gate, c) - mean, g = dnorm(c);
    q = fmaf(v, v, q), g1 += g, g2 = fmaf(g, v, g2);
  }
  const float inv = 1.f / sqrtf(block_sum(q, sh) * w + a.eps);
  g1 = a.layer ? block_sum(g1, sh) * w : 0.f;
  g2 = block_sum(g2, sh) * w * inv;
  if (threadIdx.x == 0) a.stats[blockIdx.x] = make_float4(mean, inv, g1, g2);
  for (int64_t c = c0 + threadIdx.x; c < c1; c += kThreads) {
    const float n = (after_value(a, x, gate, c) - mean) * inv;
    const float dv = norm_grad(a, inv, dnorm(c), n, g1, g2);
    if (!gate) {
      dx[c] = from_f<T>(dv);
      continue;
    }
    float f, df;
    silu_grad(to_f(gate[c]), f, df);
    if (a.inside) {
      dx[c] = from_f<T>(dv * f);
      dgate[c] = from_f<T>(dv * to_f(x[c]) * df);
    } else {
      dx[c] = from_f<T>(dv);
      const float p = fmaf(n, a.weight[c], a.bias ? a.bias[c] : 0.f);
      dgate[c] = from_f<T>(to_f(dy[c]) * (a.scale ? a.scale[c] : 1.f) * p * df);
    }
  }
}

template <class T>
__global__ void __launch_bounds__(kThreads)
norm_after_cols_kernel(NormArgs a, const T* x, const T* gate, const T* dy, float* part,
                       int64_t col_blocks, int64_t share) {
  const int64_t c = (blockIdx.x % col_blocks) * kThreads + threadIdx.x, p = blockIdx.x / col_blocks;
  if (c >= a.channels) return;
  const int64_t r1 = (p + 1) * share < a.rows ? (p + 1) * share : a.rows;
  const float w = a.weight[c], bs = a.bias ? a.bias[c] : 0.f, sc = a.scale ? a.scale[c] : 1.f;
  float dw = 0.f, db = 0.f, ds = 0.f;
  for (int64_t i = p * share; i < r1; ++i) {
    const float4 st = a.stats[i * a.groups + c / a.width];
    const T* gr = gate ? gate + i * a.gate_st : nullptr;
    const float n = (after_value(a, x + i * a.x_st, gr, c) - st.x) * st.y;
    const float o = to_f(dy[i * a.dy_st + c]);
    float f = 1.f;
    if (!a.inside && gate) {
      const float z = to_f(gr[c]);
      f = z * sigmoid_f(z);
    }
    ds = fmaf(o, fmaf(n, w, bs) * f, ds);
    dw = fmaf(o * sc * f, n, dw);
    db = fmaf(o * sc, f, db);
  }
  part[(p * 3 + 0) * a.channels + c] = dw;
  part[(p * 3 + 1) * a.channels + c] = db;
  part[(p * 3 + 2) * a.channels + c] = ds;
}

NormArgs norm_args(const ferrum_norm_args* a) {
  NormArgs n;
  n.rows = (int64_t)a->rows, n.channels = (int64_t)a->channels, n.groups = (int64_t)a->groups;
  n.width = n.channels / n.groups;
  n.eps = a->eps, n.layer = a->kind == FERRUM_NORM_LAYER, n.inside = a->gate_inside != 0;
  n.weight = a->weight, n.bias = a->bias, n.scale = a->scale;
  n.x_st = a->x_stride, n.gate_st = a->gate_stride, n.res_st = a->residual_stride;
  n.y_st = a->y_stride, n.r_st = a->r_stride, n.dy_st = a->dy_stride, n.dr_st = a->dr_stride;
  n.dx_st = a->dx_stride, n.dgate_st = a->dgate_stride, n.dres_st = a->dresidual_stride;
  n.stats = nullptr;
  return n;
}

ferrum_status check_norm(const ferrum_device* dev, const ferrum_norm_args* a, const char* what,
                         bool before, bool bwd) {
  if (ferrum_status s = check_args(dev, a, what)) return s;
  if (a->kind != FERRUM_NORM_RMS && a->kind != FERRUM_NORM_LAYER)
    return invalid(what, "kind must be FERRUM_NORM_RMS or FERRUM_NORM_LAYER");
  if (a->residual_dtype != FERRUM_F32 && a->residual_dtype != a->dtype)
    return invalid(what, "residual_dtype must be FERRUM_F32 or dtype");
  if (a->groups < 1 || a->channels % a->groups != 0 || (before && a->groups != 1))
    return invalid(what, before ? std::string("groups must be 1")
                                : "groups must divide channels (" + std::to_string(a->groups) +
                                      ", " + std::to_string(a->channels) + ")");
  if (bounded_product({a->rows, a->channels, 4}) < 0)
    return invalid(what, "rows * channels is too large");
  const size_t e = dtype_size(a->dtype), re = dtype_size(a->residual_dtype);
  const bool empty = a->rows == 0 || a->channels == 0;
  if (ferrum_status s = check_ptr(a->weight, 4, empty, what, "weight")) return s;
  if (ferrum_status s = check_ptr(a->bias, 4, true, what, "bias")) return s;
  if (ferrum_status s = check_ptr(a->scale, 4, true, what, "scale")) return s;
  if (ferrum_status s = check_ptr(a->gate, e, true, what, "gate")) return s;
  if (!bwd) {
    if (before && !empty && a->x == nullptr && a->residual == nullptr)
      return invalid(what, "x and residual are both NULL");
    if (ferrum_status s = check_ptr(a->x, e, before || empty, what, "x")) return s;
    if (ferrum_status s = check_ptr(a->residual, re, true, what, "residual")) return s;
    if (ferrum_status s = check_ptr(a->r, re, true, what, "r")) return s;
    return check_ptr(a->y, e, empty, what, "y");
  }
  if (ferrum_status s = check_ptr(a->dy, e, empty, what, "dy")) return s;
  if (ferrum_status s =
          check_ptr(a->x, e, empty || (before && a->dscale == nullptr), what, "x")) return s;
  if (before) {
    if (ferrum_status s = check_ptr(a->r, re, empty, what, "r")) return s;
    if (ferrum_status s = check_ptr(a->dr, re, true, what, "dr")) return s;
    if (ferrum_status s = check_ptr(a->dresidual, re, true, what, "dresidual")) return s;
  }
  if (ferrum_status s = check_ptr(a->dx, e, before || empty, what, "dx")) return s;
  if (ferrum_status s = check_ptr(a->dgate, e, empty || a->gate == nullptr, what, "dgate")) return s;
  if (ferrum_status s = check_ptr(a->dweight, 4, a->channels == 0, what, "dweight")) return s;
  if (ferrum_status s = check_ptr(a->dbias, 4, true, what, "dbias")) return s;
  return check_ptr(a->dscale, 4, true, what, "dscale");
}

template <class F>
ferrum_status with_residual(int dtype, int residual_dtype, F f) {
  return with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    if (residual_dtype == FERRUM_F32) return f(tag, float());
    return f(tag, T());
  });
}

// Copies the column sums to the gradients the caller asked for.
ferrum_status store_sums(const float* sums, const ferrum_norm_args* a, cudaStream_t st,
                         const char* what) {
  float* dst[3] = {a->dweight, a->dbias, a->dscale};
  for (int k = 0; k < 3; ++k)
    if (dst[k]) {
      cudaError_t e = cudaMemcpyAsync(dst[k], sums + k * a->channels, a->channels * 4,
                                      cudaMemcpyDeviceToDevice, st);
      if (e != cudaSuccess) return cuda_error(e, what);
    }
  return FERRUM_OK;
}

// Rows per block of the column sums: enough blocks to fill the GPU, and a
// workspace far below the arrays themselves.
int64_t rows_share(int64_t rows, int64_t col_blocks) {
  int64_t parts = ceil_div(148 * 4, col_blocks);
  if (parts > rows) parts = rows;
  return rows > 0 ? ceil_div(rows, parts) : 1;
}

}  // namespace
}  // namespace seq
}  // namespace ferrum

using namespace ferrum;
using namespace ferrum::seq;

extern "C" {

ferrum_status ferrum_norm_before(ferrum_device* dev, const ferrum_norm_args* a, void* stream) {
  const char* what = "norm_before";
  return guarded(what, [&]() -> ferrum_status {
    if (ferrum_status s = check_norm(dev, a, what, true, false)) return s;
    if (a->rows == 0 || a->channels == 0) return FERRUM_OK;
    if (a->rows > 0x7fffffff) return invalid(what, "too many rows for one launch");
    DeviceGuard guard(dev->ordinal);
    if (guard.status() != cudaSuccess) return cuda_error(guard.status(), "cudaSetDevice");
    return with_residual(a->dtype, a->residual_dtype, [&](auto tx, auto tr) {
      using T = decltype(tx);
      using R = decltype(tr);
      launch_detail::clear_stale_error();
      norm_before_kernel<T, R><<<(unsigned)a->rows, kThreads, 0, (cudaStream_t)stream>>>(
          norm_args(a), (const T*)a->x, (const R*)a->residual, (T*)a->y, (R*)a->r);
      return launched(what);
    });
  });
}

ferrum_status ferrum_norm_before_bwd(ferrum_device* dev, const ferrum_norm_args* a, void* stream) {
  const char* what = "norm_before_bwd";
  return guarded(what, [&]() -> ferrum_status {
    if (ferrum_status s = check_norm(dev, a, what, true, true)) return s;
    if (a->channels == 0) return FERRUM_OK;
    if (a->rows > 0x7fffffff) return invalid(what, "too many rows for one launch");
    cudaStream_t st = (cudaStream_t)stream;
    DeviceGuard guard(dev->ordinal);
    if (guard.status() != cudaSuccess) return cuda_error(guard.status(), "cudaSetDevice");
    NormArgs n = norm_args(a);
    const int64_t col_blocks = ceil_div(n.channels, kThreads);
    const int64_t share = rows_share(n.rows, col_blocks), parts = ceil_div(n.rows, share);
    PoolBuffer stats(dev, (size_t)(n.rows + 1) * sizeof(float4), st);
    PoolBuffer part(dev, (size_t)(parts + 1) * 3 * n.channels * 4, st);
    if (stats.status() != cudaSuccess) return cuda_error(stats.status(), "workspace");
    if (part.status() != cudaSuccess) return cuda_error(part.status(), "workspace");
    n.stats = stats.as<float4>();
    float* sums = part.as<float>() + parts * 3 * n.channels;
    if (n.rows > 0) {
      ferrum_status s = with_residual(a->dtype, a->residual_dtype, [&](auto tx, auto tr) {
        using T = decltype(tx);
        using R = decltype(tr);
        launch_detail::clear_stale_error();
        norm_before_bwd_kernel<T, R><<<(unsigned)n.rows, kThreads, 0, st>>>(
            n, (const R*)a->r, (const T*)a->dy, (const R*)a->dr, (T*)a->dx, (R*)a->dresidual);
        norm_before_cols_kernel<T, R><<<(unsigned)(parts * col_blocks), kThreads, 0, st>>>(
            n, a->dscale ? (const T*)a->x : nullptr, (const R*)a->r, (const T*)a->dy,
            (const R*)a->dr,
            part.as<float>(), col_blocks, share);
        return launched(what);
      });
      if (s) return s;
    }
    cudaError_t e = launch_sum_rows(part.as<float>(), parts, 3 * n.channels, sums, st);
    if (e != cudaSuccess) return cuda_error(e, what);
    return store_sums(sums, a, st, what);
  });
}

ferrum_status ferrum_norm_after(ferrum_device* dev, const ferrum_norm_args* a, void* stream) {
  const char* what = "norm_after";
  return guarded(what, [&]() -> ferrum_status {
    if (ferrum_status s = check_norm(dev, a, what, false, false)) return s;
    if (a->rows == 0 || a->channels == 0) return FERRUM_OK;
    if (a->rows * a->groups > 0x7fffffff) return invalid(what, "too many rows for one launch");
    DeviceGuard guard(dev->ordinal);
    if (guard.status() != cudaSuccess) return cuda_error(guard.status(), "cudaSetDevice");
    return with_residual(a->dtype, a->residual_dtype, [&](auto tx, auto tr) {
      using T = decltype(tx);
      using R = decltype(tr);
      launch_detail::clear_stale_error();
      norm_after_kernel<T, R>
          <<<(unsigned)(a->rows * a->groups), kThreads, 0, (cudaStream_t)stream>>>(
              norm_args(a), (const T*)a->x, (const T*)a->gate, (const R*)a->residual, (T*)a->y);
      return launched(what);
    });
  });
}

ferrum_status ferrum_norm_after_bwd(ferrum_device* dev, const ferrum_norm_args* a, void* stream) {
  const char* what = "norm_after_bwd";
  return guarded(what, [&]() -> ferrum_status {
    if (ferrum_status s = check_norm(dev, a, what, false, true)) return s;
    if (a->channels == 0) return FERRUM_OK;
    if (a->rows * a->groups > 0x7fffffff) return invalid(what, "too many rows for one launch");
    cudaStream_t st = (cudaStream_t)stream;
    DeviceGuard guard(dev->ordinal);
    if (guard.status() != cudaSuccess) return cuda_error(guard.status(), "cudaSetDevice");
    NormArgs n = norm_args(a);
    const int64_t col_blocks = ceil_div(n.channels, kThreads);
    const int64_t share = rows_share(n.rows, col_blocks), parts = ceil_div(n.rows, share);
    PoolBuffer stats(dev, (size_t)(n.rows * n.groups + 1) * sizeof(float4), st);
    PoolBuffer part(dev, (size_t)(parts + 1) * 3 * n.channels * 4, st);
    if (stats.status() != cudaSuccess) return cuda_error(stats.status(), "workspace");
    if (part.status() != cudaSuccess) return cuda_error(part.status(), "workspace");
    n.stats = stats.as<float4>();
    float* sums = part.as<float>() + parts * 3 * n.channels;
    if (n.rows > 0) {
      ferrum_status s = with_dtype(a->dtype, [&](auto tx) {
        using T = decltype(tx);
        launch_detail::clear_stale_error();
        norm_after_bwd_kernel<T><<<(unsigned)(n.rows * n.groups), kThreads, 0, st>>>(
            n, (const T*)a->x, (const T*)a->gate, (const T*)a->dy, (T*)a->dx, (T*)a->dgate);
        norm_after_cols_kernel<T><<<(unsigned)(parts * col_blocks), kThreads, 0, st>>>(
            n, (const T*)a->x, (const T*)a->gate, (const T*)a->dy, part.as<float>(), col_blocks,
            share);
        return launched(what);
      });
      if (s) return s;
    }
    cudaError_t e = launch_sum_rows(part.as<float>(), parts, 3 * n.channels, sums, st);
    if (e != cudaSuccess) return cuda_error(e, what);
    return store_sums(sums, a, st, what);
  });
}

}  // extern "C"
