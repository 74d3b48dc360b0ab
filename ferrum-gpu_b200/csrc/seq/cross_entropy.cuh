// Softmax cross entropy against a vocabulary matrix: what its translation
// units share.
#pragma once

#include <algorithm>

#include "seq_common.cuh"

namespace ferrum {
namespace seq {

__device__ __forceinline__ bool has_loss(int64_t target, int64_t vocab) {
  return target >= 0 && target < vocab;
}

// Largest value and the sum of e^(value - largest) of some of a row's logits.
// Where the largest is infinite, the sum is of e^value.
struct RowStat {
  float top, sum;
};
__device__ __forceinline__ float shift_of(float top) { return fabsf(top) == INFINITY ? 0.f : top; }
__device__ __forceinline__ RowStat join(RowStat a, RowStat b) {
  RowStat r;
  r.top = fmaxf(a.top, b.top);
  const float s = shift_of(r.top);
  const float wa = a.top == -INFINITY ? 0.f : ex2((shift_of(a.top) - s) * kLog2e);
  const float wb = b.top == -INFINITY ? 0.f : ex2((shift_of(b.top) - s) * kLog2e);
  r.sum = a.sum * wa + b.sum * wb;
  return r;
}

__device__ __forceinline__ float lse_of(RowStat r) { return shift_of(r.top) + logf(r.sum); }

// What a row needs to turn its logits into G: scaled gradients of its logits'
// sum and of its loss, lse in units of ln 2, and its target (-1 without a loss).
struct RowCoef {
  float all, one, lse2;
  int target;
};

// Lets the stream's next kernel start (where its launch allows that), and waits for
// the end of the one in front (at once where this launch did not).
__device__ __forceinline__ void start_next() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void await_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

namespace {

// ---------------------------------------------------------------- small kernels
// Each kernel of a call starts while the one in front of it ends (its barriers,
// TMEM and tensor maps are then set up already) and waits before it reads or
// writes what that one has to do with.

// 16 bytes of a row into an aligned place, zeros behind `left` values.
template <class T>
__device__ __forceinline__ void copy_unit(const T* in, int64_t left, bool wide, bool keep, T* out) {
  constexpr int kUnit = 16 / sizeof(T);
  uint4 q = make_uint4(0, 0, 0, 0);
  if (keep) {
    if (wide && left >= kUnit) {
      q = *(const uint4*)in;
    } else {
      T* e = (T*)&q;
#pragma unroll
      for (int j = 0; j < kUnit; ++j)
        if (j < left) e[j] = in[j];
    }
  }
  *(uint4*)out = q;
}

// Rows into 16-byte aligned ones of `ld` values, padded with zeros; rows without a
// loss (where targets are given) become zero. A thread copies 16 bytes.
template <class T>
__device__ void copy_rows(const T* __restrict__ in, int64_t in_ld, int64_t width, T* __restrict__ out,
                          int64_t ld, int64_t rows, const int64_t* __restrict__ targets, int64_t vocab,
                          int64_t first, int64_t stride) {
  constexpr int kUnit = 16 / sizeof(T);
  const int64_t per = ld / kUnit;
  const bool wide = in_ld % kUnit == 0 && (uintptr_t)in % 16 == 0;
  for (int64_t i = first; i < rows * per; i += stride) {
    int64_t r, c;
    if (rows * per <= 0xffffffffll) {
      r = (uint32_t)i / (uint32_t)per, c = (int64_t)((uint32_t)i % (uint32_t)per) * kUnit;
    } else {
      r = i / per, c = i % per * kUnit;
    }
    const bool keep = targets == nullptr || has_loss(targets[r], vocab);
    copy_unit(in + r * in_ld + c, width - c, wide, keep, out + r * ld + c);
  }
}

template <class T>
__global__ void __launch_bounds__(256)
copy_rows_kernel(const T* in, int64_t in_ld, int64_t width, T* out, int64_t ld, int64_t rows) {
  start_next(), await_previous();
  copy_rows<T>(in, in_ld, width, out, ld, rows, nullptr, 0, (int64_t)blockIdx.x * 256 + threadIdx.x,
               (int64_t)gridDim.x * 256);
}

// The gradient's start. The first block: scale of G and every row's coefficients;
// the others: x with rows without a loss as zeros, so that nothing of theirs
// reaches dW.
template <class T>
__global__ void __launch_bounds__(1024)
prepare_kernel(const T* x, int64_t x_ld, int64_t width, T* out, int64_t ld, int64_t tokens,
               int64_t vocab, const int64_t* __restrict__ targets, const float* __restrict__ lse,
               const float* __restrict__ dloss, const float* __restrict__ dlse,
               RowCoef* __restrict__ rows, float* scale) {
  start_next(), await_previous();
  if (blockIdx.x > 0) {
    copy_rows<T>(x, x_ld, width, out, ld, tokens, targets, vocab,
                 (int64_t)(blockIdx.x - 1) * 1024 + threadIdx.x, (int64_t)(gridDim.x - 1) * 1024);
    return;
  }
  // the largest |dloss| and |dloss + dlse|
  __shared__ float part[2][32];
  float top[2] = {0.f, 0.f};
#pragma unroll 4
  for (int64_t t = threadIdx.x; t < tokens; t += 1024) {
    const float one = dloss ? dloss[t] : 0.f, all = one + (dlse ? dlse[t] : 0.f);
    if (has_loss(targets[t], vocab)) top[0] = fmaxf(top[0], fabsf(one)), top[1] = fmaxf(top[1], fabsf(all));
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int o = 16; o > 0; o /= 2) top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
    if (threadIdx.x % 32 == 0) part[i][threadIdx.x / 32] = top[i];
  }
  __syncthreads();
  for (int i = 0; i < 32; ++i) top[0] = fmaxf(top[0], part[0][i]), top[1] = fmaxf(top[1], part[1][i]);
  // That of the loss is scaled to 2^13, unless the other is so much larger that it
  // would leave float16's range. A target's value is nearly -dloss: where all tokens
  // weigh the same it then is nearly -2^13, which 16 bits hold without the error that
  // they would all have alike. Out of the middle of the range, by a power of two;
  // 0 and infinity, not at all.
  const float unit = top[1] <= 4.f * top[0] ? top[0] : top[1];
  float up = 8192.f / unit, down = unit / 8192.f;
  if (!(unit > 0x1p-100f && unit < 0x1p100f)) {
    const int e = (__float_as_int(unit) >> 23) - 127;
    const int s = e == -127 || e == 128 ? 0 : (13 - e > 126 ? 126 : (13 - e < -126 ? -126 : 13 - e));
    up = __int_as_float((127 + s) << 23), down = __int_as_float((127 - s) << 23);
  }
  if (threadIdx.x == 0) scale[0] = up, scale[1] = down;
#pragma unroll 4
  for (int64_t t = threadIdx.x; t < tokens; t += 1024) {
    const int64_t at = targets[t];
    const float one = dloss ? dloss[t] : 0.f, all = one + (dlse ? dlse[t] : 0.f);
    const float norm = lse[t] * kLog2e;
    const bool counts = has_loss(at, vocab);
    rows[t] = {counts ? all * up : 0.f, counts ? one * up : 0.f, counts ? norm : 0.f,
               counts ? (int)at : -1};
  }
}

// dx from the slabs of its sums, in their order; 4 values a thread.
template <class T>
__global__ void __launch_bounds__(256)
finish_dx_kernel(const float* __restrict__ sums, int splits, int64_t ld, int64_t tokens,
                 int64_t width, const RowCoef* __restrict__ rows, const float* __restrict__ scale,
                 T* __restrict__ dx, int64_t dx_ld) {
  await_previous();
  const float inv = scale[1];
  const int64_t per = ld / 4;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < tokens * per; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per, c = i % per * 4;
    const bool keep = rows[r].target >= 0;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int s = 0; s < splits; ++s) {
      const float4 u = *(const float4*)(sums + ((int64_t)s * tokens + r) * ld + c);
      v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
    }
    const float o[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c + j < width) dx[r * dx_ld + c + j] = from_f<T>(keep ? o[j] * inv : 0.f);
  }
}

// A launch that may start while the call's one in front of it ends (`first`: one that
// may not).
template <class... P, class... A>
ferrum_status start(const char* what, bool first, void (*kernel)(P...), int64_t grid, int block,
                    size_t smem, cudaStream_t stream, A... args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid), cfg.blockDim = dim3((unsigned)block);
  cfg.dynamicSmemBytes = smem, cfg.stream = stream, cfg.attrs = attr, cfg.numAttrs = first ? 0 : 1;
  launch_detail::clear_stale_error();
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  return e == cudaSuccess ? FERRUM_OK : cuda_error(e, what);
}

// An operand as the products need it: the caller's array, or a copy in 16-byte rows.
template <class T>
struct Matrix {
  const T* p;
  int64_t ld;
};
inline int64_t padded(int64_t n) { return ceil_div(n, 8) * 8; }

template <class T>
ferrum_status copied(Matrix<T>& m, int64_t width, int64_t rows, uint8_t*& at, bool first,
                     cudaStream_t stream, const char* what) {
  const int64_t ld = padded(width);
  const ferrum_status s =
      start(what, first, copy_rows_kernel<T>, std::min<int64_t>(ceil_div(rows * ld / 8, 256), 148 * 32),
            256, 0, stream, m.p, m.ld, width, (T*)at, ld, rows);
  m = {(const T*)at, ld};
  at += rows * ld * (int64_t)sizeof(T);
  return s;
}

}  // namespace

// A row's loss and lse from `parts` statistics of each row.
ferrum_status finish_loss(const RowStat* stats, int parts, const float* at_target,
                          const ferrum_cross_entropy_args* a, cudaStream_t stream, const char* what);

ferrum_status loss_fwd_f32(ferrum_device* dev, const ferrum_cross_entropy_args* a,
                           cudaStream_t stream, const char* what);
ferrum_status loss_bwd_f32(ferrum_device* dev, const ferrum_cross_entropy_args* a,
                           cudaStream_t stream, const char* what);
ferrum_status loss_fwd_tc(ferrum_device* dev, const ferrum_cross_entropy_args* a,
                          cudaStream_t stream, const char* what);
ferrum_status loss_bwd_tc(ferrum_device* dev, const ferrum_cross_entropy_args* a,
                          cudaStream_t stream, const char* what);

}  // namespace seq
}  // namespace ferrum
