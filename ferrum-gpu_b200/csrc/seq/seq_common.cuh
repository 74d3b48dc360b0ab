// Shared pieces of the sequence operators (include/ferrum_seq.h): element
// types, the activation functions, reductions, and the host-side argument
// checks, workspaces and error handling of their C entry points.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <exception>
#include <new>
#include <string>
#include <type_traits>

#include "../../../include/ferrum_seq.h"
#include "../launch_common.cuh"
#include "../runtime.h"

namespace ferrum {
namespace seq {

using launch_detail::ceil_div;

// ---------------------------------------------------------------- device
template <class T>
__device__ __forceinline__ float to_f(T v) { return (float)v; }
template <>
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }

template <class T>
__device__ __forceinline__ T from_f(float v) { return (T)v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

constexpr float kLog2e = 1.4426950408889634f;

// 2^x by the special-function unit (2 units in the last place).
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// 1 / x by the special-function unit (1 unit in the last place).
__device__ __forceinline__ float rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// 1 / (1 + e^-x). For x below about -88 e^-x overflows to infinity, whose
// reciprocal is 0, the limit.
__device__ __forceinline__ float sigmoid_f(float x) { return rcp(1.f + ex2(-x * kLog2e)); }

// Two 16-bit values rounded and packed by one instruction.
template <class T>
__device__ __forceinline__ uint32_t pack_pair(float x, float y) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(x, y);
    return *(const uint32_t*)&h;
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *(const uint32_t*)&h;
  }
}

// VL consecutive values to and from float32 in accesses of up to 16 bytes (the
// caller has checked the alignment); single values for VL = 1.
template <class T, int VL>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[VL]) {
  if constexpr (VL == 1) {
    v[0] = to_f(*p);
  } else if constexpr (sizeof(T) == 4 && VL == 2) {
    const float2 u = *(const float2*)p;
    v[0] = u.x, v[1] = u.y;
  } else if constexpr (VL == 2) {
    const uint32_t u = *(const uint32_t*)p;
    const T* w = (const T*)&u;
    v[0] = to_f(w[0]), v[1] = to_f(w[1]);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < VL; i += 4) {
      const float4 u = *(const float4*)(p + i);
      v[i] = u.x, v[i + 1] = u.y, v[i + 2] = u.z, v[i + 3] = u.w;
    }
  } else if constexpr (VL == 4) {
    const uint2 u = *(const uint2*)p;
    const T* w = (const T*)&u;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = to_f(w[i]);
  } else {
    const uint4 u = *(const uint4*)p;
    const T* w = (const T*)&u;
#pragma unroll
    for (int i = 0; i < VL; ++i) v[i] = to_f(w[i]);
  }
}
template <class T, int VL>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[VL]) {
  if constexpr (VL == 1) {
    *p = from_f<T>(v[0]);
  } else if constexpr (sizeof(T) == 4 && VL == 2) {
    *(float2*)p = make_float2(v[0], v[1]);
  } else if constexpr (VL == 2) {
    *(uint32_t*)p = pack_pair<T>(v[0], v[1]);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < VL; i += 4) *(float4*)(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
  } else {
    uint32_t w[VL / 2];
#pragma unroll
    for (int i = 0; i < VL / 2; ++i) w[i] = pack_pair<T>(v[2 * i], v[2 * i + 1]);
    if constexpr (VL == 4)
      *(uint2*)p = *(const uint2*)w;
    else
      *(uint4*)p = *(const uint4*)w;
  }
}

// Asynchronous copies from global to shared memory, `bytes` of the unit read
// and the rest zeroed.
template <int UNIT>
__device__ __forceinline__ void cp_async(void* dst, const void* src, int bytes) {
  const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
  if constexpr (UNIT == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(src), "r"(bytes));
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(d), "l"(src), "r"(bytes));
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;"); }
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Sum over the 32 lanes, in every lane, in a fixed order.
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// ---------------------------------------------------------------- host
// A (batch, length, channels) argument with its element type.
template <class T>
struct Rows {
  T* p;
  int64_t sb, st;
  __device__ __forceinline__ T* at(int64_t b, int64_t t) const { return p + b * sb + t * st; }
  __host__ __device__ explicit operator bool() const { return p != nullptr; }
};
template <class T>
Rows<T> rows_of(const ferrum_rows& r) { return Rows<T>{(T*)r.ptr, r.batch_stride, r.row_stride}; }

inline size_t dtype_size(int dtype) { return dtype == FERRUM_F32 ? 4 : 2; }

// Workspace from the device's stream-ordered pool, returned to it on scope
// exit (in stream order, so after the work enqueued in between).
class PoolBuffer {
 public:
  PoolBuffer(ferrum_device* dev, size_t bytes, cudaStream_t stream) : stream_(stream) {
    if (bytes > 0) status_ = cudaMallocFromPoolAsync(&p_, bytes, dev->pool, stream);
  }
  ~PoolBuffer() {
    if (p_) (void)cudaFreeAsync(p_, stream_);
  }
  PoolBuffer(const PoolBuffer&) = delete;
  PoolBuffer& operator=(const PoolBuffer&) = delete;
  cudaError_t status() const { return status_; }
  template <class T>
  T* as() const { return (T*)p_; }

 private:
  void* p_ = nullptr;
  cudaStream_t stream_;
  cudaError_t status_ = cudaSuccess;
};

inline ferrum_status invalid(const char* what, const std::string& msg) {
  return set_error(FERRUM_ERR_INVALID_ARG, std::string(what) + ": " + msg);
}

inline bool aligned(const void* p, size_t n) { return ((uintptr_t)p % n) == 0; }

// Common checks of an entry point: handle, argument block, element type.
template <class Args>
ferrum_status check_args(const ferrum_device* dev, const Args* a, const char* what) {
  if (dev == nullptr || dev->tables == nullptr)
    return set_error(FERRUM_ERR_INVALID_ARG, "device handle is NULL or destroyed");
  if (a == nullptr) return invalid(what, "args is NULL");
  if (a->struct_size != sizeof(Args))
    return invalid(what, "struct_size is " + std::to_string(a->struct_size) + ", expected " +
                             std::to_string(sizeof(Args)));
  if (a->dtype != FERRUM_F32 && a->dtype != FERRUM_F16 && a->dtype != FERRUM_BF16)
    return invalid(what, "dtype must be FERRUM_F32, FERRUM_F16 or FERRUM_BF16, got " +
                             std::to_string(a->dtype));
  return FERRUM_OK;
}

// An array argument: present (unless `optional`) and aligned to its element.
inline ferrum_status check_ptr(const void* p, size_t align, bool optional, const char* what,
                               const char* name) {
  if (p == nullptr) {
    if (optional) return FERRUM_OK;
    return invalid(what, std::string(name) + " is NULL");
  }
  if (!aligned(p, align))
    return invalid(what, std::string(name) + " must be " + std::to_string(align) + "-byte aligned");
  return FERRUM_OK;
}

// Most values one array of a call may hold, as for the transforms.
constexpr int64_t kMaxElems = (int64_t)1 << kMaxLogElems;

// product of sizes, or -1 above kMaxElems
inline int64_t bounded_product(std::initializer_list<size_t> f) {
  int64_t p = 1;
  for (size_t v : f) {
    if (v == 0) return 0;
    if (v > (size_t)kMaxElems || p > kMaxElems / (int64_t)v) return -1;
    p *= (int64_t)v;
  }
  return p;
}

// Runs a C entry's body: makes the device current, and turns anything the
// body throws into a status (nothing may unwind through a C caller).
template <class F>
ferrum_status guarded(const char* what, F body) noexcept {
  try {
    clear_error();
    return body();
  } catch (const std::bad_alloc&) {
    try {
      return set_error(FERRUM_ERR_ALLOC, std::string(what) + ": out of host memory");
    } catch (...) {
      return FERRUM_ERR_ALLOC;
    }
  } catch (const std::exception& e) {
    try {
      return set_error(FERRUM_ERR_CUDA, std::string(what) + ": " + e.what());
    } catch (...) {
      return FERRUM_ERR_CUDA;
    }
  } catch (...) {
    return FERRUM_ERR_CUDA;
  }
}

inline ferrum_status launched(const char* what) {
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? FERRUM_OK : cuda_error(e, what);
}

// Calls f with a value of the element type `dtype` names.
template <class F>
ferrum_status with_dtype(int dtype, F f) {
  if (dtype == FERRUM_F32) return f(float());
  if (dtype == FERRUM_F16) return f(__half());
  return f(__nv_bfloat16());
}

// Sums over r < rows of part[r * n + i], in a fixed order (results do not
// depend on scheduling): to out[i] for i < split, to rest[i - split] (where
// rest is given) for the others.
cudaError_t launch_sum_rows(const float* part, int64_t rows, int64_t n, int64_t split, float* out,
                            float* rest, cudaStream_t stream);

}  // namespace seq
}  // namespace ferrum
