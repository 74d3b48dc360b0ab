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

// |value| from which on its multiple by log2 e may leave float32's range: the difference is
// taken first then.
constexpr float kFar = 2e38f;

__device__ __forceinline__ float lse_of(RowStat r) { return shift_of(r.top) + logf(r.sum); }

// What a row needs to turn its logits into G: scaled gradients of its logits'
// sum and of its loss, lse, and its target (-1 without a loss).
struct RowCoef {
  float all, one, lse;
  int target;
};
// softmax = 2^(logit scale - lse scale). Where lse is finite and beyond kFar, logits are 2^104
// and more apart, or equal: any scale serves that keeps the products finite.
__device__ __forceinline__ float softmax_scale(float lse) {
  return fabsf(lse) > kFar && fabsf(lse) < INFINITY ? 0x1p-30f : kLog2e;
}

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

// 16 bytes of a row, zeros behind `left` values.
template <class T>
__device__ __forceinline__ uint4 row_unit(const T* in, int64_t left, bool wide) {
  constexpr int kUnit = 16 / sizeof(T);
  if (wide && left >= kUnit) return *(const uint4*)in;
  uint4 q = make_uint4(0, 0, 0, 0);
  T* e = (T*)&q;
#pragma unroll
  for (int j = 0; j < kUnit; ++j)
    if (j < left) e[j] = in[j];
  return q;
}

// Rows into 16-byte aligned ones of `ld` values, padded with zeros. A thread copies 16
// bytes at a time.
template <class T>
__global__ void __launch_bounds__(256)
copy_rows_kernel(const T* __restrict__ in, int64_t in_ld, int64_t width, T* __restrict__ out, int64_t ld,
                 int64_t rows) {
  start_next(), await_previous();
  constexpr int kUnit = 16 / sizeof(T);
  const int64_t per = ld / kUnit;
  const bool wide = in_ld % kUnit == 0 && (uintptr_t)in % 16 == 0;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * per; i += (int64_t)gridDim.x * 256) {
    int64_t r, c;
    if (rows * per <= 0xffffffffll) {
      r = (uint32_t)i / (uint32_t)per, c = (int64_t)((uint32_t)i % (uint32_t)per) * kUnit;
    } else {
      r = i / per, c = i % per * kUnit;
    }
    *(uint4*)(out + r * ld + c) = row_unit(in + r * in_ld + c, width - c, wide);
  }
}

// The gradient works on the tokens that have a loss, one after the other, as many as
// there are rounded up to `round` (and that many at least), whole steps of a product's
// depth: the rows behind the last are zeros.
struct LiveTokens {
  RowCoef* rows;             // coefficients
  int* index;                // their place among all tokens; -1 behind the last
  int* count;                // with those behind the last
  float* scale;              // of G, and its inverse
  int round;                 // 64 at most
  int64_t x_rows;            // rows of x that exist: none behind them is read
};

// The gradient's start: the tokens with a loss moved together (x into 16-byte rows of
// `ld` values), scale of G and every row's coefficients, dx of the others zeroed. Each
// block counts the tokens in front of its own.
template <class T>
__global__ void __launch_bounds__(1024)
prepare_kernel(const T* __restrict__ x, int64_t x_ld, int64_t width, T* __restrict__ out, int64_t ld,
               int64_t tokens, int64_t vocab, const int64_t* __restrict__ targets,
               const float* __restrict__ lse, const float* __restrict__ dloss,
               const float* __restrict__ dlse, LiveTokens live, T* __restrict__ dx, int64_t dx_ld) {
  constexpr int kUnit = 16 / sizeof(T);
  __shared__ float part[2][32];
  __shared__ int counts[2][32], place[1024];
  start_next(), await_previous();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t each = (tokens + gridDim.x - 1) / gridDim.x, r0 = blockIdx.x * each;
  const int64_t r1 = r0 + each < tokens ? r0 + each : tokens;
  // the largest |dloss| and |dloss + dlse|, tokens in front of the block's, all tokens
  float top[2] = {0.f, 0.f};
  int n[2] = {0, 0};
#pragma unroll 4
  for (int64_t t = threadIdx.x; t < tokens; t += 1024) {
    const float one = dloss ? dloss[t] : 0.f, all = one + (dlse ? dlse[t] : 0.f);
    if (has_loss(targets[t], vocab)) {
      top[0] = fmaxf(top[0], fabsf(one)), top[1] = fmaxf(top[1], fabsf(all));
      n[0] += t < r0, n[1] += 1;
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int o = 16; o > 0; o /= 2) {
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
      n[i] += __shfl_xor_sync(0xffffffffu, n[i], o);
    }
    if (lane == 0) part[i][warp] = top[i], counts[i][warp] = n[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    top[i] = part[i][lane], n[i] = counts[i][lane];
#pragma unroll
    for (int o = 16; o > 0; o /= 2) {
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
      n[i] += __shfl_xor_sync(0xffffffffu, n[i], o);
    }
  }
  const int total = n[1];
  const int padded_total = total > 0 ? (total + live.round - 1) / live.round * live.round : live.round;
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
  if (blockIdx.x == 0 && threadIdx.x == 0) live.scale[0] = up, live.scale[1] = down, *live.count = padded_total;
  const int64_t per = ld / kUnit;
  const bool wide = x_ld % kUnit == 0 && (uintptr_t)x % 16 == 0;
  const bool wide_dx = dx_ld % kUnit == 0 && (uintptr_t)dx % 16 == 0;
  int next = n[0];                       // place of the next token with a loss
  for (int64_t base = r0; base < r1; base += 1024) {
    const int64_t t = base + threadIdx.x;
    const int64_t at = t < r1 ? targets[t] : -1;
    const bool counts_for = t < r1 && has_loss(at, vocab);
    const uint32_t mask = __ballot_sync(0xffffffffu, counts_for);
    __syncthreads();                     // (what the turn before read)
    if (lane == 0) counts[0][warp] = __popc(mask);
    __syncthreads();
    int in_front = lane < warp ? counts[0][lane] : 0, group = counts[0][lane];
#pragma unroll
    for (int o = 16; o > 0; o /= 2) {
      in_front += __shfl_xor_sync(0xffffffffu, in_front, o);
      group += __shfl_xor_sync(0xffffffffu, group, o);
    }
    const int mine = next + in_front + __popc(mask & ((1u << lane) - 1));
    next += group;
    place[threadIdx.x] = counts_for ? mine : -1;
    if (counts_for) {
      const float one = dloss ? dloss[t] : 0.f, all = one + (dlse ? dlse[t] : 0.f);
      live.rows[mine] = {all * up, one * up, lse[t], (int)at};
      live.index[mine] = (int)t;
    }
    __syncthreads();
    const int rows = r1 - base < 1024 ? (int)(r1 - base) : 1024;
    // a warp a row, four loads of a lane under way at once
    for (int r = warp; r < rows; r += 32) {
      const int to = place[r];
      if (to >= 0) {
        const T* from = x + (base + r) * x_ld;
        for (int64_t u = lane; u < per; u += 128) {
          uint4 q[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (u + 32 * j < per) q[j] = row_unit(from + (u + 32 * j) * kUnit, width - (u + 32 * j) * kUnit, wide);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (u + 32 * j < per) *(uint4*)(out + to * ld + (u + 32 * j) * kUnit) = q[j];
        }
      } else {
        T* zero = dx + (base + r) * dx_ld;
        for (int64_t c = lane * kUnit; c < width; c += 32 * kUnit) {
          if (wide_dx && c + kUnit <= width) {
            *(uint4*)(zero + c) = make_uint4(0, 0, 0, 0);
          } else {
            for (int j = 0; j < kUnit && c + j < width; ++j) zero[c + j] = from_f<T>(0.f);
          }
        }
      }
    }
  }
  if (blockIdx.x == gridDim.x - 1) {
    const int behind = padded_total - total;
    if ((int)threadIdx.x < behind) {
      live.rows[total + threadIdx.x] = {0.f, 0.f, 0.f, -1};
      live.index[total + threadIdx.x] = -1;
    }
    const int64_t zeros = (padded_total < live.x_rows ? padded_total : live.x_rows) - total;
    for (int64_t i = threadIdx.x; i < zeros * per; i += 1024)
      *(uint4*)(out + total * ld + i * kUnit) = make_uint4(0, 0, 0, 0);
  }
}

// dx from the slabs of its sums, of `rows` rows each, in their order; 4 values a thread.
template <class T>
__global__ void __launch_bounds__(256)
finish_dx_kernel(const float* __restrict__ sums, int splits, int64_t ld, int64_t rows, int64_t width,
                 LiveTokens live, T* __restrict__ dx, int64_t dx_ld) {
  await_previous();
  const float inv = live.scale[1];
  const int64_t per = ld / 4, all = *live.count * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int64_t r = all <= 0xffffffffll ? (uint32_t)i / (uint32_t)per : i / per, c = (i - r * per) * 4;
    const int at = live.index[r];
    if (at < 0) continue;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int s = 0; s < splits; ++s) {
      const float4 u = *(const float4*)(sums + ((int64_t)s * rows + r) * ld + c);
      v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
    }
    const float o[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c + j < width) dx[at * dx_ld + c + j] = from_f<T>(o[j] * inv);
  }
}

// Tokens of each split of dW's depth, whole steps of it; splits behind the last have none.
__host__ __device__ inline int64_t live_each(int64_t live, int splits, int step) {
  return ((live + step - 1) / step + splits - 1) / splits * step;
}

// dW from the slabs of its sums, of `words` rows each, in their order; 4 values a thread.
template <class T>
__global__ void __launch_bounds__(256)
finish_dw_kernel(const float* __restrict__ sums, int splits, int step, int64_t ld, int64_t words,
                 int64_t width, LiveTokens live, T* __restrict__ dw, int64_t dw_ld) {
  await_previous();
  const float inv = live.scale[1];
  const int64_t each = live_each(*live.count, splits, step), per = ld / 4, all = words * per;
  const int used = (int)((*live.count + each - 1) / each);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int64_t r = all <= 0xffffffffll ? (uint32_t)i / (uint32_t)per : i / per, c = (i - r * per) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int s = 0; s < used; ++s) {
      const float4 u = *(const float4*)(sums + ((int64_t)s * words + r) * ld + c);
      v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
    }
    const float o[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c + j < width) dw[r * dw_ld + c + j] = from_f<T>(o[j] * inv);
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
// SMs of the current device.
inline int sm_count() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    sms = 148;
  return sms;
}
// Blocks of the gradient's start: a token and 16 KiB of x each at least, and no more than run at
// once, since each looks through all targets for those in front of its own.
inline int64_t blocks_to_prepare(int64_t tokens, int64_t bytes) {
  return std::max<int64_t>(1, std::min({ceil_div(tokens * bytes, 16 * 1024), tokens, (int64_t)sm_count() * 2}));
}
inline int64_t padded(int64_t n) { return ceil_div(n, 8) * 8; }

template <class T>
ferrum_status copied(Matrix<T>& m, int64_t width, int64_t rows, uint8_t*& at, bool first,
                     cudaStream_t stream, const char* what) {
  const int64_t ld = padded(width);
  const ferrum_status s =
      start(what, first, copy_rows_kernel<T>, std::min<int64_t>(ceil_div(rows * ld / 8, 256), sm_count() * 32),
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
