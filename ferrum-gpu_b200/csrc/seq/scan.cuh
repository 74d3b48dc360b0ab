// Argument views and helpers shared by the selective scan's kernels.
#pragma once

#include <cfloat>
#include <type_traits>

#include "seq_common.cuh"

namespace ferrum {
namespace seq {

constexpr int kSaveSteps = FERRUM_SCAN_SAVE_STEPS;

struct ScanSizes {
  int64_t batch, length, channels, groups, per_group, saves;
  int states;
  bool softplus;
};

template <class T>
struct ScanIn {
  Rows<T> u, delta, z, B, C;
  int64_t B_group, C_group;
  const float *A, *D, *bias;
  const float* initial;
  const int32_t* lengths;
};

__device__ __forceinline__ int64_t scan_length(const int32_t* lengths, int64_t b, int64_t length) {
  if (lengths == nullptr) return length;
  const int64_t n = lengths[b];
  return n < 0 ? 0 : (n > length ? length : n);
}

// The smaller value, or NaN where either is one.
__device__ __forceinline__ float min_nan(float x, float y) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}

// e^-|x|, flushed to 0 below 2^-126 (|x| above 87.3). 2^t takes t with a
// rounding error of up to |t| 2^-24, 64 units of the result at |x| = 87; what
// the product |x| log2 e loses, d, is put back as e (1 + d ln 2).
__device__ __forceinline__ float exp_minus(float x) {
  const float ax = -min_nan(fabsf(x), 200.f), t = ax * kLog2e;   // (finite: inf - inf is NaN)
  const float d = fmaf(ax, kLog2e, -t);
  const float e = ex2(t);
  return fmaf(e, fmaf(ax, 1.3349758e-8f, d * 0.69314718f), e);   // 1.33e-8 = ln 2 (log2 e - kLog2e)
}

// log(1 + e^x) = max(x, 0) + log(1 + e), e = e^-|x| in (0, 1]. log(1 + e) / e
// is a polynomial in e (least squares at Chebyshev nodes of [0, 1], relative
// error 6.1e-8), so small results keep their relative accuracy (9 units of
// 2^-24 in all, down to x = -87); it costs one exponential and a dozen products
// and sums, where log1pf takes a few times that and the scan spends it once
// per value.
__device__ __forceinline__ float softplus_of(float x, float e) {
  float p = 0.00525345793f;
  p = fmaf(p, e, -0.0295885075f);
  p = fmaf(p, e, 0.0783616677f);
  p = fmaf(p, e, -0.136747703f);
  p = fmaf(p, e, 0.191114306f);
  p = fmaf(p, e, -0.248443693f);
  p = fmaf(p, e, 0.333192706f);
  p = fmaf(p, e, -0.499995023f);
  p = fmaf(p, e, 1.f);
  return fmaf(p, e, fmaxf(x, 0.f));
}
__device__ __forceinline__ float softplus_f(float x) { return softplus_of(x, exp_minus(x)); }
// The same, and its slope 1 / (1 + e^-x).
__device__ __forceinline__ float softplus_f(float x, float& slope) {
  const float e = exp_minus(x), r = rcp(1.f + e);
  slope = x < 0.f ? e * r : r;
  return softplus_of(x, e);
}

// Pairs of floats for the two-wide FP32 instructions.
using f2 = unsigned long long;
__device__ __forceinline__ f2 pack(float x, float y) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 unpack(f2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// A state's rate A as the kernels take it, for factors 2^(dt A log2 e). An
// infinite one becomes the largest float, so that steps of dt = 0, which fill
// up a sequence's last piece, leave the state as it is (0 * inf would be NaN);
// any other step still takes the factor to 0.
__device__ __forceinline__ float scaled_rate(float A) {
  const float r = A * kLog2e;
  return isinf(r) ? copysignf(FLT_MAX, r) : r;
}

// Added to the exponent of a step's factor, in the product's multiply-add. The
// special-function unit's 2^x errs to one side: measured over -1 < x < -2^-8 by
// -0.3 to -0.45 units of 2^-24 on average, which adds up where a state keeps
// its value over many steps. With half a unit more the average is within 0.1 of zero there
// (0.26 closer to 1), and 2^0 is still 1. Over 400 steps with dt |A| from 0.001
// to 0.16 the state is 1.6e-7 from its 64-bit value and dA 5e-7 (1.5e-6 and
// 3.7e-6 without; a plain float32 loop 3.2e-7 and 6.6e-7), in the same time.
constexpr float kExponentShift = 0x1p-25f;
__device__ __forceinline__ f2 exponents(f2 dt, f2 A) {
  return fma2(dt, A, pack(kExponentShift, kExponentShift));
}

// A piece of a (steps, columns) array in shared memory, in its own type: row
// t at t * COLS elements plus 16 bytes for every 8 rows, so that lanes 8 rows
// apart meet different banks.
template <class T, int COLS>
struct Piece {
  static constexpr int SKEW = 16 / (int)sizeof(T);
  __host__ __device__ static constexpr int size(int rows) { return rows * COLS + rows / 8 * SKEW; }
  __device__ static __forceinline__ int at(int t, int c) { return t * COLS + (t >> 3) * SKEW + c; }
};

// How the rows of a call's arrays can be copied: 16 bytes or 4 bytes at a
// time, or (0) by single elements where a row starts at an odd element.
enum { kCopyScalar = 0, kCopy4 = 4, kCopy16 = 16 };

template <class T>
int copy_unit(const ferrum_rows& r, int64_t extra = 0) {
  const uintptr_t v = (uintptr_t)r.ptr | (uintptr_t)(r.batch_stride * (int64_t)sizeof(T)) |
                      (uintptr_t)(r.row_stride * (int64_t)sizeof(T)) |
                      (uintptr_t)(extra * (int64_t)sizeof(T));
  return v % 16 == 0 ? kCopy16 : (v % 4 == 0 ? kCopy4 : kCopyScalar);
}

// Rows [0, ROWS) of columns [0, cols) of an array to a piece, rows from
// `rows` and columns from `cols` on as zeros. THREADS threads take part; the
// 16- and 4-byte forms are asynchronous. Row strides fit 32 bits (checked on
// the host), so an address is one wide multiply-add.
template <class T, int ROWS, int COLS, int THREADS, int UNIT>
__device__ __forceinline__ void copy_units(T* dst, const T* src, int stride, int rows, int cols,
                                           int tid) {
  constexpr int E = UNIT / (int)sizeof(T), PER = COLS / E;
#pragma unroll
  for (int i0 = 0; i0 < ROWS * PER; i0 += THREADS) {
    const int i = i0 + tid;
    if (ROWS * PER % THREADS != 0 && i >= ROWS * PER) break;
    const int t = i / PER, c = (i % PER) * E;
    int n = t < rows ? cols - c : 0;
    n = n < 0 ? 0 : (n > E ? E : n);
    cp_async<UNIT>(dst + Piece<T, COLS>::at(t, c), n > 0 ? src + (int64_t)t * stride + c : src,
                   n * (int)sizeof(T));
  }
}
template <class T, int ROWS, int COLS, int THREADS>
__device__ __forceinline__ void copy_piece(T* dst, const T* src, int stride, int rows, int cols,
                                           int unit, int tid) {
  if constexpr (COLS * sizeof(T) >= 16) {
    if (unit == kCopy16) return copy_units<T, ROWS, COLS, THREADS, 16>(dst, src, stride, rows, cols, tid);
  }
  if (unit != kCopyScalar)
    return copy_units<T, ROWS, COLS, THREADS, 4>(dst, src, stride, rows, cols, tid);
  for (int i = tid; i < ROWS * COLS; i += THREADS) {
    const int t = i / COLS, c = i % COLS;
    dst[Piece<T, COLS>::at(t, c)] =
        (t < rows && c < cols) ? src[(int64_t)t * stride + c] : from_f<T>(0.f);
  }
}

// A piece in shared memory to rows [0, rows), columns [0, cols) of an array.
template <class T, int ROWS, int COLS, int THREADS>
__device__ __forceinline__ void store_piece(T* dst, const T* src, int stride, int rows, int cols,
                                            int unit, int tid) {
  if constexpr (COLS * sizeof(T) >= 16) {
    if (unit == kCopy16 && cols == COLS) {
      constexpr int E = 16 / (int)sizeof(T), PER = COLS / E;
#pragma unroll
      for (int i0 = 0; i0 < ROWS * PER; i0 += THREADS) {
        const int i = i0 + tid, t = i / PER, c = (i % PER) * E;
        if (i < ROWS * PER && t < rows)
          *(uint4*)(dst + (int64_t)t * stride + c) = *(const uint4*)(src + Piece<T, COLS>::at(t, c));
      }
      return;
    }
  }
#pragma unroll 4
  for (int i = tid; i < ROWS * COLS; i += THREADS) {
    const int t = i / COLS, c = i % COLS;
    if (t < rows && c < cols) dst[(int64_t)t * stride + c] = src[Piece<T, COLS>::at(t, c)];
  }
}

// A piece of rows [0, ROWS) converted to float32, two values at a time.
template <class T, int ROWS, int COLS, int THREADS>
__device__ __forceinline__ void widen_piece(float* dst, const T* src, int tid) {
#pragma unroll
  for (int i0 = 0; i0 < ROWS * COLS / 2; i0 += THREADS) {
    const int i = i0 + tid;
    if (ROWS * COLS / 2 % THREADS != 0 && i >= ROWS * COLS / 2) break;
    const int t = i / (COLS / 2), c = i % (COLS / 2) * 2;
    float2 v;
    if constexpr (std::is_same<T, float>::value)
      v = *(const float2*)(src + Piece<T, COLS>::at(t, c));
    else if constexpr (std::is_same<T, __half>::value)
      v = __half22float2(*(const __half2*)(src + Piece<T, COLS>::at(t, c)));
    else
      v = __bfloat1622float2(*(const __nv_bfloat162*)(src + Piece<T, COLS>::at(t, c)));
    *(float2*)(dst + Piece<float, COLS>::at(t, c)) = v;
  }
}

template <class T>
ScanIn<T> scan_in(const ferrum_scan_args* a) {
  return ScanIn<T>{rows_of<T>(a->u), rows_of<T>(a->delta), rows_of<T>(a->z), rows_of<T>(a->B),
                   rows_of<T>(a->C), a->B_group_stride, a->C_group_stride, a->A, a->D,
                   a->delta_bias, a->initial_state, a->lengths};
}

ferrum_status check_scan(const ferrum_device* dev, const ferrum_scan_args* a, const char* what,
                         bool bwd);

inline ScanSizes scan_sizes(const ferrum_scan_args* a) {
  ScanSizes s;
  s.batch = (int64_t)a->batch, s.length = (int64_t)a->length, s.channels = (int64_t)a->channels;
  s.groups = (int64_t)a->groups, s.per_group = s.channels / s.groups;
  s.saves = ceil_div(s.length, kSaveSteps);
  s.states = (int)a->states, s.softplus = a->delta_softplus != 0;
  return s;
}

template <class F>
ferrum_status with_states(int n, F f) {
  if (n <= 8) return f(std::integral_constant<int, 8>());
  if (n <= 16) return f(std::integral_constant<int, 16>());
  if (n <= 32) return f(std::integral_constant<int, 32>());
  return f(std::integral_constant<int, 64>());
}

}  // namespace seq
}  // namespace ferrum
