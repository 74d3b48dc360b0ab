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
// A few operations per moved value, so HBM bounds it: every array is read and
// written once. A row (behind: a group of one) stays in the registers of a
// warp, or of a block of 128 to 1024 threads for wide rows, in 16-byte
// accesses where the arrays allow. The gradient kernel also keeps the column
// sums (dweight, dbias, dscale) of all the rows that a warp or block takes, so
// no second pass over the arrays is needed; their few hundred partial sums
// are added in a fixed order.
// Measured, bf16, of the 6.5 TB/s of a copy: norm_before with a float32 residual,
// 16384 x 2048, 69 us (90 %), its gradient 139 us (66 %; waits on loads at 32
// warps an SM); norm_after, 8191 x 4096 in 8 groups, 69 us (60 %) and 111 us
// (46 %): issue slots (58 and 68 %) and the gate's two special functions. In one
// group (512 threads a row) 78 and 166 us: barriers, and in the gradient the
// column sums' spills, which above 8192 values cost most of the time
// (4000 x 12000: 141 and 658 us; norm_before's gradient 350).
#include <algorithm>

#include "seq_common.cuh"

namespace ferrum {
namespace seq {
namespace {

constexpr int64_t kMaxWidth = 32768;

struct NormArgs {
  int64_t rows, channels, groups, width;  // width = channels / groups
  float eps;
  bool layer;
  const float *weight, *bias, *scale;
  int64_t x_st, gate_st, res_st, y_st, r_st, dy_st, dr_st, dx_st, dgate_st, dres_st;
};

// Sums of N values over the TPR threads of a row, in every thread, in a fixed
// order. Blocks alternate between two buffers: one barrier per call.
template <int TPR, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* sh, int& flip) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
  if constexpr (TPR > 32) {
    constexpr int W = TPR / 32;
    float* buf = sh + flip * W * 3;
    flip ^= 1;
    const int w = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) buf[i * W + w] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (W <= 4) {
        float s = buf[i * W];
#pragma unroll
        for (int k = 1; k < W; ++k) s += buf[i * W + k];
        v[i] = s;
      } else {
        v[i] = warp_sum((threadIdx.x & 31) < W ? buf[i * W + (threadIdx.x & 31)] : 0.f);
      }
    }
  }
}

// The rows of one warp or block ("unit"): its group, its lane in the row.
template <int TPR, int VL, int NC>
struct Unit {
  static constexpr int THREADS = TPR == 32 ? 256 : TPR;
  int64_t index, count, g, first, step;
  int lane;
  __device__ __forceinline__ Unit(int64_t groups) {
    // for a whole block the row is uniform, and so are its addresses
    index = TPR == THREADS ? blockIdx.x
                           : ((int64_t)blockIdx.x * THREADS + threadIdx.x) / TPR;
    count = (int64_t)gridDim.x * (THREADS / TPR);
    g = index % groups, first = index / groups, step = count / groups;
    if (index >= step * groups) first = INT64_MAX;   // units beyond a multiple of the groups
    lane = threadIdx.x % TPR;
  }
  // column of chunk k in the group, and whether it lies in it
  __device__ __forceinline__ int col(int k) const { return (k * TPR + lane) * VL; }
};

// Warps an SM that the registers must allow for, so that enough loads are in
// flight: 32; in norm_after's gradient, which spills more than it gains there,
// 24 for blocks of up to 256 threads (us with 24 and 32: 16384 x 2048 in 8 groups
// 111, 123, in one 138, 156; 65536 x 512 121, 140; 200000 x 128 170, 191). Wider
// blocks lose by it (8191 x 4096 in one group 178, 166).
constexpr int kWarps = 32, kAfterBwdWarps = 24;
constexpr int min_blocks(int tpr, int values, int warps) {
  return values > 8 ? 1 : (tpr == 32 ? warps / 8 : std::max(1, warps * 32 / tpr));
}
constexpr int after_bwd_warps(int tpr) { return tpr <= 256 ? kAfterBwdWarps : kWarps; }

// The next row's line to the L2 cache while this row is worked on: 8 % for
// norm_before at 8191 x 4096; the other kernels, bound by instructions, lose.
template <class T>
__device__ __forceinline__ void prefetch(const T* p) {
  asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
}

// Gradient of a value from that of its normalised value n.
__device__ __forceinline__ float norm_grad(const NormArgs& a, float inv, float dn, float n,
                                           float mean_dn, float mean_dnn) {
  if (a.width == 1) return a.layer ? 0.f : inv * dn * (a.eps * inv * inv);
  return inv * (dn - mean_dn - n * mean_dnn);
}

// d silu(g) / dg, and silu(g)
__device__ __forceinline__ void silu_grad(float g, float& f, float& df) {
  const float sg = sigmoid_f(g);
  f = g * sg;
  df = sg * (1.f + g * (1.f - sg));
}

// The mean of a row held as v (zeros beyond its end): 0 for RMS.
template <int TPR, int VL, int NC>
__device__ __forceinline__ float row_mean(const NormArgs& a, const float (&v)[NC][VL], float* sh,
                                          int& flip) {
  if (!a.layer) return 0.f;
  float q[1] = {0.f};
#pragma unroll
  for (int k = 0; k < NC; ++k)
#pragma unroll
    for (int e = 0; e < VL; ++e) q[0] += v[k][e];
  row_sum<TPR>(q, sh, flip);
  return q[0] / (float)a.width;
}

// mean and 1 / deviation of a row held as v
template <int TPR, int VL, int NC>
__device__ __forceinline__ void row_stats(const NormArgs& a, const Unit<TPR, VL, NC>& u,
                                          const float (&v)[NC][VL], float& mean, float& inv,
                                          float* sh, int& flip) {
  const float w = 1.f / (float)a.width;
  mean = row_mean<TPR>(a, v, sh, flip);
  float q[1];
  q[0] = 0.f;
#pragma unroll
  for (int k = 0; k < NC; ++k)
    if (u.col(k) < a.width)
#pragma unroll
      for (int e = 0; e < VL; ++e) q[0] = fmaf(v[k][e] - mean, v[k][e] - mean, q[0]);
  row_sum<TPR>(q, sh, flip);
  inv = 1.f / sqrtf(fmaf(q[0], w, a.eps));
}

// VL floats of a parameter, or a constant where it is absent
template <int VL>
__device__ __forceinline__ void load_param(const float* p, int64_t c, float (&v)[VL], float other) {
  if (p) {
    load_vec<float, VL>(p + c, v);
  } else {
#pragma unroll
    for (int e = 0; e < VL; ++e) v[e] = other;
  }
}

template <class T, class R, int TPR, int VL, int NC>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR, min_blocks(TPR, VL * NC, kWarps))
norm_before_kernel(NormArgs a, const T* x, const R* res, T* y, R* r) {
  __shared__ float sh[2 * 3 * TPR / 32];
  const Unit<TPR, VL, NC> u(a.groups);
  int flip = 0;
  for (int64_t row = u.first; row < a.rows; row += u.step) {
    if (row + u.step < a.rows)
#pragma unroll
      for (int k = 0; k < NC; ++k)
        if (u.col(k) < a.width) {
          if (x) prefetch(x + (row + u.step) * a.x_st + u.col(k));
          if (res) prefetch(res + (row + u.step) * a.res_st + u.col(k));
        }
    float v[NC][VL];
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = u.col(k);
#pragma unroll
      for (int e = 0; e < VL; ++e) v[k][e] = 0.f;
      if (c >= a.width) continue;
      if (res) load_vec<R, VL>(res + row * a.res_st + c, v[k]);
      if (x) {
        float xv[VL], sc[VL];
        load_vec<T, VL>(x + row * a.x_st + c, xv);
        load_param<VL>(a.scale, c, sc, 1.f);
#pragma unroll
        for (int e = 0; e < VL; ++e) v[k][e] = fmaf(sc[e], xv[e], v[k][e]);
      }
      if (r) store_vec<R, VL>(r + row * a.r_st + c, v[k]);
    }
    float mean, inv;
    row_stats(a, u, v, mean, inv, sh, flip);
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = u.col(k);
      if (c >= a.width) continue;
      float w[VL], bs[VL];
      load_vec<float, VL>(a.weight + c, w);
      load_param<VL>(a.bias, c, bs, 0.f);
#pragma unroll
      for (int e = 0; e < VL; ++e) v[k][e] = fmaf((v[k][e] - mean) * inv, w[e], bs[e]);
      store_vec<T, VL>(y + row * a.y_st + c, v[k]);
    }
  }
}

// A unit's column sums to part[(unit * 3 + j) * width + column].
template <int TPR, int VL, int NC>
__device__ __forceinline__ void store_sums(const NormArgs& a, const Unit<TPR, VL, NC>& u,
                                           const float (&s)[3][NC][VL], float* part) {
#pragma unroll
  for (int j = 0; j < 3; ++j)
#pragma unroll
    for (int k = 0; k < NC; ++k)
      if (u.col(k) < a.width)
#pragma unroll
        for (int e = 0; e < VL; ++e) part[(u.index * 3 + j) * a.width + u.col(k) + e] = s[j][k][e];
}

template <class T, class R, bool BIAS, int TPR, int VL, int NC>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR, min_blocks(TPR, VL * NC, kWarps))
norm_before_bwd_kernel(NormArgs a, const T* x, const R* r, const T* dy, const R* dr, T* dx, R* dres,
                       float* part) {
  __shared__ float sh[2 * 3 * TPR / 32];
  const Unit<TPR, VL, NC> u(a.groups);
  int flip = 0;
  float sums[3][NC][VL] = {};      // dweight, dbias, dscale
  const float w1 = 1.f / (float)a.width;
  for (int64_t row = u.first; row < a.rows; row += u.step) {
    float v[NC][VL], g[NC][VL], dn[NC][VL];   // r (then centred), dy, gradient of n
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = u.col(k);
#pragma unroll
      for (int e = 0; e < VL; ++e) v[k][e] = 0.f, g[k][e] = 0.f;
      if (c >= a.width) continue;
      load_vec<R, VL>(r + row * a.r_st + c, v[k]);
      load_vec<T, VL>(dy + row * a.dy_st + c, g[k]);
    }
    const float mean = row_mean<TPR>(a, v, sh, flip);
    float m[3] = {0.f, 0.f, 0.f};             // sums of v^2, dn and dn * v
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = u.col(k);
      if (c >= a.width) continue;
      float w[VL];
      load_vec<float, VL>(a.weight + c, w);
#pragma unroll
      for (int e = 0; e < VL; ++e) {
        v[k][e] -= mean;
        dn[k][e] = g[k][e] * w[e];
        m[0] = fmaf(v[k][e], v[k][e], m[0]);
        m[1] += dn[k][e];
        m[2] = fmaf(dn[k][e], v[k][e], m[2]);
      }
    }
    row_sum<TPR>(m, sh, flip);
    const float inv = 1.f / sqrtf(fmaf(m[0], w1, a.eps));
    const float g1 = a.layer ? m[1] * w1 : 0.f, g2 = m[2] * inv * w1;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = u.col(k);
      if (c >= a.width) continue;
      float o[VL];
#pragma unroll
      for (int e = 0; e < VL; ++e) {
        const float n = v[k][e] * inv;
        sums[0][k][e] = fmaf(g[k][e], n, sums[0][k][e]);
        if constexpr (BIAS) sums[1][k][e] += g[k][e];
        o[e] = norm_grad(a, inv, dn[k][e], n, g1, g2);
      }
      if (dr) {
        float q[VL];
        load_vec<R, VL>(dr + row * a.dr_st + c, q);
#pragma unroll
        for (int e = 0; e < VL; ++e) o[e] += q[e];
      }
      if (dres) store_vec<R, VL>(dres + row * a.dres_st + c, o);
      if (x) {                     // dscale is wanted
        float q[VL];
        load_vec<T, VL>(x + row * a.x_st + c, q);
#pragma unroll
        for (int e = 0; e < VL; ++e) sums[2][k][e] = fmaf(o[e], q[e], sums[2][k][e]);
      }
      if (dx) {
        float sc[VL];
        load_param<VL>(a.scale, c, sc, 1.f);
#pragma unroll
        for (int e = 0; e < VL; ++e) o[e] *= sc[e];
        store_vec<T, VL>(dx + row * a.dx_st + c, o);
      }
    }
  }
  store_sums(a, u, sums, part);
}

// Where the gate enters.
enum { kNoGate = 0, kInside = 1, kOutside = 2 };

template <class T, class R, int GATE, int TPR, int VL, int NC>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR, min_blocks(TPR, VL * NC, kWarps))
norm_after_kernel(NormArgs a, const T* x, const T* gate, const R* res, T* y) {
  __shared__ float sh[2 * 3 * TPR / 32];
  const Unit<TPR, VL, NC> u(a.groups);
  int flip = 0;
  const int64_t off = u.g * a.width;
  for (int64_t row = u.first; row < a.rows; row += u.step) {
    float v[NC][VL], f[NC][VL];    // the norm's input; silu(gate) where it comes after
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int64_t c = off + u.col(k);
#pragma unroll
      for (int e = 0; e < VL; ++e) v[k][e] = 0.f, f[k][e] = 1.f;
      if (u.col(k) >= a.width) continue;
      load_vec<T, VL>(x + row * a.x_st + c, v[k]);
      if constexpr (GATE != kNoGate) {
        load_vec<T, VL>(gate + row * a.gate_st + c, f[k]);
#pragma unroll
        for (int e = 0; e < VL; ++e) {
          f[k][e] *= sigmoid_f(f[k][e]);
          if constexpr (GATE == kInside) v[k][e] *= f[k][e], f[k][e] = 1.f;
        }
      }
    }
    float mean, inv;
    row_stats(a, u, v, mean, inv, sh, flip);
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int64_t c = off + u.col(k);
      if (u.col(k) >= a.width) continue;
      float w[VL], bs[VL], sc[VL], base[VL];
      load_vec<float, VL>(a.weight + c, w);
      load_param<VL>(a.bias, c, bs, 0.f);
      load_param<VL>(a.scale, c, sc, 1.f);
#pragma unroll
      for (int e = 0; e < VL; ++e) base[e] = 0.f;
      if (res) load_vec<R, VL>(res + row * a.res_st + c, base);
#pragma unroll
      for (int e = 0; e < VL; ++e) {
        const float p = fmaf((v[k][e] - mean) * inv, w[e], bs[e]) * f[k][e];
        base[e] = fmaf(sc[e], p, base[e]);
      }
      store_vec<T, VL>(y + row * a.y_st + c, base);
    }
  }
}

template <class T, int GATE, int TPR, int VL, int NC>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR,
                                  min_blocks(TPR, VL * NC, after_bwd_warps(TPR)))
norm_after_bwd_kernel(NormArgs a, const T* x, const T* gate, const T* dy, T* dx, T* dgate,
                      float* part) {
  __shared__ float sh[2 * 3 * TPR / 32];
  const Unit<TPR, VL, NC> u(a.groups);
  int flip = 0;
  const int64_t off = u.g * a.width;
  float sums[3][NC][VL] = {};      // dweight, dbias, dscale
  const float w1 = 1.f / (float)a.width;
  for (int64_t row = u.first; row < a.rows; row += u.step) {
    float v[NC][VL], z[NC][VL], o[NC][VL];   // norm input (then n), gate, dy (then dn)
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int64_t c = off + u.col(k);
#pragma unroll
      for (int e = 0; e < VL; ++e) v[k][e] = 0.f, z[k][e] = 0.f, o[k][e] = 0.f;
      if (u.col(k) >= a.width) continue;
      load_vec<T, VL>(x + row * a.x_st + c, v[k]);
      load_vec<T, VL>(dy + row * a.dy_st + c, o[k]);
      if constexpr (GATE != kNoGate) {
        load_vec<T, VL>(gate + row * a.gate_st + c, z[k]);
        if constexpr (GATE == kInside)
#pragma unroll
          for (int e = 0; e < VL; ++e) v[k][e] *= z[k][e] * sigmoid_f(z[k][e]);
      }
    }
    float mean, inv;
    row_stats(a, u, v, mean, inv, sh, flip);
    float m[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int64_t c = off + u.col(k);
      if (u.col(k) >= a.width) continue;
      float w[VL], bs[VL], sc[VL], dg[VL];
      load_vec<float, VL>(a.weight + c, w);
      load_param<VL>(a.bias, c, bs, 0.f);
      load_param<VL>(a.scale, c, sc, 1.f);
#pragma unroll
      for (int e = 0; e < VL; ++e) {
        const float n = (v[k][e] - mean) * inv, p = fmaf(n, w[e], bs[e]);
        float f = 1.f, df = 0.f;
        if constexpr (GATE == kOutside) silu_grad(z[k][e], f, df);
        sums[2][k][e] = fmaf(o[k][e], p * f, sums[2][k][e]);
        const float g = o[k][e] * sc[e];
        dg[e] = g * p * df;
        sums[0][k][e] = fmaf(g * f, n, sums[0][k][e]);
        sums[1][k][e] = fmaf(g, f, sums[1][k][e]);
        v[k][e] = n;
        o[k][e] = g * f * w[e];
        m[0] += o[k][e], m[1] = fmaf(o[k][e], n, m[1]);
      }
      if constexpr (GATE == kOutside) store_vec<T, VL>(dgate + row * a.dgate_st + c, dg);
    }
    row_sum<TPR>(m, sh, flip);
    const float g1 = a.layer ? m[0] * w1 : 0.f, g2 = m[1] * w1;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int64_t c = off + u.col(k);
      if (u.col(k) >= a.width) continue;
#pragma unroll
      for (int e = 0; e < VL; ++e) o[k][e] = norm_grad(a, inv, o[k][e], v[k][e], g1, g2);
      if constexpr (GATE == kInside) {
        float xv[VL], dg[VL];
        load_vec<T, VL>(x + row * a.x_st + c, xv);   // again, from the cache
#pragma unroll
        for (int e = 0; e < VL; ++e) {
          float f, df;
          silu_grad(z[k][e], f, df);
          dg[e] = o[k][e] * xv[e] * df;
          o[k][e] *= f;
        }
        store_vec<T, VL>(dgate + row * a.dgate_st + c, dg);
      }
      store_vec<T, VL>(dx + row * a.dx_st + c, o[k]);
    }
  }
  store_sums(a, u, sums, part);
}

// The units' column sums, added in a fixed order: unit j * groups + g holds
// group g's. 32 columns by 32 strands of units.
__global__ void __launch_bounds__(1024)
norm_sums_kernel(const float* __restrict__ part, int64_t units, int64_t groups, int64_t width,
                 float* dweight, float* dbias, float* dscale) {
  __shared__ float sh[32][33];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int64_t wb = (width + 31) / 32;
  int64_t q = blockIdx.x;
  const int64_t i0 = q % wb * 32;
  q /= wb;
  const int64_t g = q % groups;
  const int k = (int)(q / groups);
  float* out = k == 0 ? dweight : (k == 1 ? dbias : dscale);
  if (out == nullptr) return;
  float s = 0.f;
  if (i0 + x < width) {
#pragma unroll 4
    for (int64_t j = y; j < units / groups; j += 32)
      s += part[((j * groups + g) * 3 + k) * width + i0 + x];
  }
  sh[y][x] = s;
  __syncthreads();
  s = warp_sum(sh[x][y]);       // column y of the 32, over the strands
  if (x == 0 && i0 + y < width) out[g * width + i0 + y] = s;
}

NormArgs norm_args(const ferrum_norm_args* a) {
  NormArgs n;
  n.rows = (int64_t)a->rows, n.channels = (int64_t)a->channels, n.groups = (int64_t)a->groups;
  n.width = n.channels / n.groups;
  n.eps = a->eps, n.layer = a->kind == FERRUM_NORM_LAYER;
  n.weight = a->weight, n.bias = a->bias, n.scale = a->scale;
  n.x_st = a->x_stride, n.gate_st = a->gate_stride, n.res_st = a->residual_stride;
  n.y_st = a->y_stride, n.r_st = a->r_stride, n.dy_st = a->dy_stride, n.dr_st = a->dr_stride;
  n.dx_st = a->dx_stride, n.dgate_st = a->dgate_stride, n.dres_st = a->dresidual_stride;
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
  if ((int64_t)(a->channels / a->groups) > kMaxWidth)
    return invalid(what, "a normalised row may have at most 32768 values, got " +
                             std::to_string(a->channels / a->groups));
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

// Threads per row, values per access and accesses per thread for a row of
// `width` values: f(TPR, VL, NC) with TPR * VL * NC >= width. 8 values a
// thread up to width 8192: few registers, many warps.
template <int V>
using Int = std::integral_constant<int, V>;
template <class F>
ferrum_status with_shape(int64_t width, bool vec, F f) {
  if (vec) {
    if (width <= 256) return f(Int<32>(), Int<8>(), Int<1>());
    if (width <= 512) return f(Int<64>(), Int<8>(), Int<1>());
    if (width <= 1024) return f(Int<128>(), Int<8>(), Int<1>());
    if (width <= 2048) return f(Int<256>(), Int<8>(), Int<1>());
    if (width <= 4096) return f(Int<512>(), Int<8>(), Int<1>());
    if (width <= 8192) return f(Int<1024>(), Int<8>(), Int<1>());
    return f(Int<1024>(), Int<8>(), Int<4>());
  }
  if (width <= 256) return f(Int<32>(), Int<1>(), Int<8>());
  if (width <= 2048) return f(Int<256>(), Int<1>(), Int<8>());
  if (width <= 8192) return f(Int<1024>(), Int<1>(), Int<8>());
  return f(Int<1024>(), Int<1>(), Int<32>());
}
template <class F>
void with_gate(const ferrum_norm_args* a, F f) {
  if (a->gate == nullptr) return f(Int<kNoGate>());
  if (a->gate_inside) return f(Int<kInside>());
  return f(Int<kOutside>());
}

// Whether rows can go in 16-byte accesses.
bool rows_vec(const void* p, int64_t stride, size_t e) {
  return p == nullptr || (aligned(p, 16) && (stride * (int64_t)e) % 16 == 0);
}
bool norm_vec(const ferrum_norm_args* a, bool bwd) {
  const size_t e = dtype_size(a->dtype), re = dtype_size(a->residual_dtype);
  const int64_t width = (int64_t)(a->channels / a->groups);
  bool v = width % 8 == 0 && rows_vec(a->weight, 0, 4) && rows_vec(a->bias, 0, 4) &&
           rows_vec(a->scale, 0, 4) && rows_vec(a->x, a->x_stride, e) &&
           rows_vec(a->gate, a->gate_stride, e) && rows_vec(a->r, a->r_stride, re);
  if (!bwd) return v && rows_vec(a->residual, a->residual_stride, re) && rows_vec(a->y, a->y_stride, e);
  return v && rows_vec(a->dy, a->dy_stride, e) && rows_vec(a->dr, a->dr_stride, re) &&
         rows_vec(a->dx, a->dx_stride, e) && rows_vec(a->dgate, a->dgate_stride, e) &&
         rows_vec(a->dresidual, a->dresidual_stride, re);
}

// Blocks of a launch: enough units for all rows, at most `per_sm` blocks' worth
// of threads on every SM, and a number of units that holds every group.
template <int TPR>
int64_t unit_blocks(int64_t rows, int64_t groups, int threads_per_sm) {
  constexpr int threads = TPR == 32 ? 256 : TPR, per = threads / TPR;
  int64_t blocks = std::min(ceil_div(rows * groups, per),
                            (int64_t)148 * std::max(1, threads_per_sm / threads));
  const int64_t need = ceil_div(groups, per);
  return std::max(blocks, need);
}

}  // namespace
}  // namespace seq
}  // namespace ferrum

using namespace ferrum;
using namespace ferrum::seq;

namespace {

template <class Go>
ferrum_status norm_fwd(ferrum_device* dev, const ferrum_norm_args* a, bool before,
                       const char* what, Go go) {
  if (ferrum_status s = check_norm(dev, a, what, before, false)) return s;
  if (a->rows == 0 || a->channels == 0) return FERRUM_OK;
  DeviceGuard guard(dev->ordinal);
  if (guard.status() != cudaSuccess) return cuda_error(guard.status(), "cudaSetDevice");
  const NormArgs n = norm_args(a);
  return with_residual(a->dtype, a->residual_dtype, [&](auto tx, auto tr) {
    return with_shape(n.width, norm_vec(a, false), [&](auto tpr, auto vl, auto nc) {
      constexpr int TPR = decltype(tpr)::value;
      const int64_t blocks = unit_blocks<TPR>(n.rows, n.groups, kWarps * 32);
      launch_detail::clear_stale_error();
      go(n, tx, tr, tpr, vl, nc, (unsigned)blocks, TPR == 32 ? 256 : TPR);
      return launched(what);
    });
  });
}

// The gradients' launch and the sums of its units.
template <class Go>
ferrum_status norm_bwd(ferrum_device* dev, const ferrum_norm_args* a, bool before,
                       const char* what, cudaStream_t st, Go go) {
  if (ferrum_status s = check_norm(dev, a, what, before, true)) return s;
  if (a->channels == 0) return FERRUM_OK;
  DeviceGuard guard(dev->ordinal);
  if (guard.status() != cudaSuccess) return cuda_error(guard.status(), "cudaSetDevice");
  const NormArgs n = norm_args(a);
  return with_residual(a->dtype, a->residual_dtype, [&](auto tx, auto tr) {
    return with_shape(n.width, norm_vec(a, true), [&](auto tpr, auto vl, auto nc) -> ferrum_status {
      constexpr int TPR = decltype(tpr)::value;
      constexpr int threads = TPR == 32 ? 256 : TPR;
      const int64_t blocks = unit_blocks<TPR>(
          n.rows, n.groups, 32 * (before ? kWarps : after_bwd_warps(TPR)));
      const int64_t units = blocks * (threads / TPR) / n.groups * n.groups;
      PoolBuffer part(dev, sizeof(float) * (size_t)(blocks * (threads / TPR) * 3 * n.width), st);
      if (part.status() != cudaSuccess) return cuda_error(part.status(), "workspace");
      launch_detail::clear_stale_error();
      go(n, tx, tr, tpr, vl, nc, (unsigned)blocks, threads, part.as<float>());
      norm_sums_kernel<<<(unsigned)(ceil_div(n.width, 32) * n.groups * 3), 1024, 0, st>>>(
          part.as<float>(), units, n.groups, n.width, a->dweight, a->dbias, a->dscale);
      return launched(what);
    });
  });
}

}  // namespace

extern "C" {

ferrum_status ferrum_norm_before(ferrum_device* dev, const ferrum_norm_args* a, void* stream) {
  const char* what = "norm_before";
  return guarded(what, [&]() -> ferrum_status {
    return norm_fwd(dev, a, true, what, [&](const NormArgs& n, auto tx, auto tr, auto tpr, auto vl,
                                            auto nc, unsigned blocks, int threads) {
      using T = decltype(tx);
      using R = decltype(tr);
      norm_before_kernel<T, R, decltype(tpr)::value, decltype(vl)::value, decltype(nc)::value>
          <<<blocks, threads, 0, (cudaStream_t)stream>>>(n, (const T*)a->x, (const R*)a->residual,
                                                         (T*)a->y, (R*)a->r);
    });
  });
}

ferrum_status ferrum_norm_before_bwd(ferrum_device* dev, const ferrum_norm_args* a, void* stream) {
  const char* what = "norm_before_bwd";
  return guarded(what, [&]() -> ferrum_status {
    return norm_bwd(dev, a, true, what, (cudaStream_t)stream,
                    [&](const NormArgs& n, auto tx, auto tr, auto tpr, auto vl, auto nc,
                        unsigned blocks, int threads, float* part) {
      using T = decltype(tx);
      using R = decltype(tr);
      auto go = [&](auto bias) {
        norm_before_bwd_kernel<T, R, decltype(bias)::value, decltype(tpr)::value,
                               decltype(vl)::value, decltype(nc)::value>
            <<<blocks, threads, 0, (cudaStream_t)stream>>>(
                n, a->dscale ? (const T*)a->x : nullptr, (const R*)a->r, (const T*)a->dy,
                (const R*)a->dr, (T*)a->dx, (R*)a->dresidual, part);
      };
      if (a->dbias)     // its sums take registers that the others can use
        go(std::true_type());
      else
        go(std::false_type());
    });
  });
}

ferrum_status ferrum_norm_after(ferrum_device* dev, const ferrum_norm_args* a, void* stream) {
  const char* what = "norm_after";
  return guarded(what, [&]() -> ferrum_status {
    return norm_fwd(dev, a, false, what, [&](const NormArgs& n, auto tx, auto tr, auto tpr, auto vl,
                                             auto nc, unsigned blocks, int threads) {
      using T = decltype(tx);
      using R = decltype(tr);
      with_gate(a, [&](auto gate) {
        norm_after_kernel<T, R, decltype(gate)::value, decltype(tpr)::value, decltype(vl)::value,
                          decltype(nc)::value><<<blocks, threads, 0, (cudaStream_t)stream>>>(
            n, (const T*)a->x, (const T*)a->gate, (const R*)a->residual, (T*)a->y);
      });
    });
  });
}

ferrum_status ferrum_norm_after_bwd(ferrum_device* dev, const ferrum_norm_args* a, void* stream) {
  const char* what = "norm_after_bwd";
  return guarded(what, [&]() -> ferrum_status {
    return norm_bwd(dev, a, false, what, (cudaStream_t)stream,
                    [&](const NormArgs& n, auto tx, auto, auto tpr, auto vl, auto nc,
                        unsigned blocks, int threads, float* part) {
      using T = decltype(tx);
      with_gate(a, [&](auto gate) {
        norm_after_bwd_kernel<T, decltype(gate)::value, decltype(tpr)::value, decltype(vl)::value,
                              decltype(nc)::value><<<blocks, threads, 0, (cudaStream_t)stream>>>(
            n, (const T*)a->x, (const T*)a->gate, (const T*)a->dy, (T*)a->dx, (T*)a->dgate, part);
      });
    });
  });
}

}  // extern "C"
