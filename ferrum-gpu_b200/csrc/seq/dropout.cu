// Dropout from a counter-based generator, added onto a residual:
//   y = residual + (word(i) >= p 2^32 ? x / (1 - p) : 0)
// word(i) is word i % 4 of Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel
// random numbers: as easy as 1, 2, 3", SC 2011) of counter (i / 4, offset) and key
// seed. Element i's word depends on nothing else, so no mask is stored, the
// gradient draws the same words, and neither strides nor the launch change them.
// A dropped value is selected away, not multiplied: an infinity or NaN there
// leaves no trace.
//
// A thread takes 8 adjacent elements: two counters, 16-byte accesses. Contiguous
// arrays are one row, whatever their shape.
#include <type_traits>

#include "seq_common.cuh"

namespace ferrum {
namespace seq {
namespace {

constexpr int kThreads = 256;
constexpr int kVec = 8;

struct Draw {
  uint64_t seed, offset;
  const uint64_t* seed_ptr;
  uint32_t least;      // words below it are dropped
  float scale;
  bool none;           // p = 1: nothing is kept
};

struct Words {
  uint32_t w[4];
};
__device__ __forceinline__ Words philox(uint64_t counter, uint64_t offset, uint64_t key) {
  uint32_t c0 = (uint32_t)counter, c1 = (uint32_t)(counter >> 32);
  uint32_t c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
  uint32_t k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0, c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
    c1 = (uint32_t)p1, c3 = (uint32_t)p0;
    k0 += 0x9E3779B9u, k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

__device__ __forceinline__ float drop(uint32_t word, float x, float res, const Draw& d) {
  return word >= d.least && !d.none ? fmaf(x, d.scale, res) : res;
}

// y = res + dropout(x). FLAT: one row (rows = 1). Threads run over groups of
// kVec elements of a row; VEC says that all rows can be accessed a group at a
// time, which also means that a group starts at a multiple of 8 elements.
template <class T, class R, bool VEC, bool FLAT>
__global__ void __launch_bounds__(kThreads)
dropout_kernel(const T* __restrict__ x, const R* __restrict__ res, R* __restrict__ y,
               int64_t x_stride, int64_t res_stride, int64_t y_stride, int64_t channels,
               int64_t per_row, int64_t groups, Draw d) {
  const int64_t g = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (g >= groups) return;
  int64_t row = 0, col = g;
  if constexpr (!FLAT) {
    if (groups <= 0xffffffffll) {
      row = (uint32_t)g / (uint32_t)per_row, col = (uint32_t)g % (uint32_t)per_row;
    } else {
      row = g / per_row, col = g % per_row;
    }
  }
  col *= kVec;
  const uint64_t first = (uint64_t)(row * channels + col);
  const uint64_t key = d.seed_ptr ? *d.seed_ptr : d.seed;
  x += row * x_stride + col, y += row * y_stride + col;
  if (res) res += row * res_stride + col;
  if (VEC && col + kVec <= channels) {
    float v[kVec], o[kVec];
    load_vec<T, kVec>(x, v);
    if (res) {
      load_vec<R, kVec>(res, o);
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i) o[i] = 0.f;
    }
#pragma unroll
    for (int q = 0; q < kVec / 4; ++q) {
      const Words w = philox(first / 4 + q, d.offset, key);
#pragma unroll
      for (int i = 0; i < 4; ++i) o[4 * q + i] = drop(w.w[i], v[4 * q + i], o[4 * q + i], d);
    }
    store_vec<R, kVec>(y, o);
    return;
  }
  // single elements: the end of a row, or rows that are not aligned
  const int n = channels - col < kVec ? (int)(channels - col) : kVec;
  uint64_t have = ~0ull;
  Words w = {};
  for (int i = 0; i < n; ++i) {
    const uint64_t e = first + i;
    if (e / 4 != have) have = e / 4, w = philox(have, d.offset, key);
    const uint32_t k = (uint32_t)e % 4;
    const uint32_t word = k < 2 ? (k == 0 ? w.w[0] : w.w[1]) : (k == 2 ? w.w[2] : w.w[3]);
    y[i] = from_f<R>(drop(word, to_f(x[i]), res ? to_f(res[i]) : 0.f, d));
  }
}

template <class T, class R>
ferrum_status launch(const void* x, const void* res, void* y, int64_t xs, int64_t rs, int64_t ys,
                     int64_t rows, int64_t channels, const Draw& d, cudaStream_t stream,
                     const char* what) {
  const bool flat =
      rows == 1 || (xs == channels && ys == channels && (res == nullptr || rs == channels));
  if (flat) channels *= rows, rows = 1;
  auto ok = [&](const void* p, int64_t stride, size_t e) {
    return aligned(p, 16) && (flat || stride * (int64_t)e % 16 == 0);
  };
  const bool vec = ok(x, xs, sizeof(T)) && ok(y, ys, sizeof(R)) &&
                   (res == nullptr || ok(res, rs, sizeof(R))) && (flat || channels % kVec == 0);
  const int64_t per_row = ceil_div(channels, kVec), groups = rows * per_row;
  const int64_t blocks = ceil_div(groups, kThreads);
  if (blocks > 0x7fffffff) return invalid(what, "too many values for one launch");
  auto run = [&](auto v, auto f) {
    launch_detail::clear_stale_error();
    dropout_kernel<T, R, decltype(v)::value, decltype(f)::value>
        <<<(unsigned)blocks, kThreads, 0, stream>>>((const T*)x, (const R*)res, (R*)y, xs, rs, ys,
                                                    channels, per_row, groups, d);
    return launched(what);
  };
  using Y = std::true_type;
  using N = std::false_type;
  if (flat) return vec ? run(Y(), Y()) : run(N(), Y());
  return vec ? run(Y(), N()) : run(N(), N());
}

ferrum_status check_dropout(const ferrum_device* dev, const ferrum_dropout_args* a, const char* what,
                            bool bwd) {
  if (ferrum_status s = check_args(dev, a, what)) return s;
  if (a->residual_dtype != FERRUM_F32 && a->residual_dtype != a->dtype)
    return invalid(what, "residual_dtype must be FERRUM_F32 or dtype, got " +
                             std::to_string(a->residual_dtype));
  if (!(a->p >= 0.0 && a->p <= 1.0)) return invalid(what, "p must be in [0, 1], got " + std::to_string(a->p));
  if (bounded_product({a->rows, a->channels}) < 0) return invalid(what, "rows * channels is too large");
  const bool empty = a->rows == 0 || a->channels == 0;
  const size_t e = dtype_size(a->dtype), r = dtype_size(a->residual_dtype);
  if (ferrum_status s = check_ptr(a->seed_ptr, 8, true, what, "seed_ptr")) return s;
  if (bwd) {
    if (ferrum_status s = check_ptr(a->dy, r, empty, what, "dy")) return s;
    return check_ptr(a->dx, e, empty, what, "dx");
  }
  if (ferrum_status s = check_ptr(a->x, e, empty, what, "x")) return s;
  if (ferrum_status s = check_ptr(a->residual, r, true, what, "residual")) return s;
  return check_ptr(a->y, r, empty, what, "y");
}

Draw draw_of(const ferrum_dropout_args* a) {
  Draw d = {};
  d.seed = a->seed, d.offset = a->offset, d.seed_ptr = a->seed_ptr;
  d.none = a->p == 1.0;
  d.least = d.none ? 0xffffffffu : (uint32_t)(a->p * 4294967296.0);
  d.scale = d.none ? 0.f : (float)(1.0 / (1.0 - a->p));
  return d;
}

}  // namespace
}  // namespace seq
}  // namespace ferrum

using namespace ferrum;
using namespace ferrum::seq;

extern "C" {

ferrum_status ferrum_dropout(ferrum_device* dev, const ferrum_dropout_args* a, void* stream) {
  const char* what = "dropout";
  return guarded(what, [&]() -> ferrum_status {
    if (ferrum_status s = check_dropout(dev, a, what, false)) return s;
    if (a->rows == 0 || a->channels == 0) return FERRUM_OK;
    DeviceGuard guard(dev->ordinal);
    if (guard.status() != cudaSuccess) return cuda_error(guard.status(), "cudaSetDevice");
    return with_dtype(a->dtype, [&](auto tag) {
      using T = decltype(tag);
      auto go = [&](auto r) {
        return launch<T, decltype(r)>(a->x, a->residual, a->y, a->x_stride, a->residual_stride,
                                      a->y_stride, (int64_t)a->rows, (int64_t)a->channels,
                                      draw_of(a), (cudaStream_t)stream, what);
      };
      return a->residual_dtype == FERRUM_F32 ? go(float()) : go(T());
    });
  });
}

ferrum_status ferrum_dropout_bwd(ferrum_device* dev, const ferrum_dropout_args* a, void* stream) {
  const char* what = "dropout_bwd";
  return guarded(what, [&]() -> ferrum_status {
    if (ferrum_status s = check_dropout(dev, a, what, true)) return s;
    if (a->rows == 0 || a->channels == 0) return FERRUM_OK;
    DeviceGuard guard(dev->ordinal);
    if (guard.status() != cudaSuccess) return cuda_error(guard.status(), "cudaSetDevice");
    return with_dtype(a->dtype, [&](auto tag) {
      using T = decltype(tag);
      auto go = [&](auto r) {
        return launch<decltype(r), T>(a->dy, nullptr, a->dx, a->dy_stride, 0, a->dx_stride,
                                      (int64_t)a->rows, (int64_t)a->channels, draw_of(a),
                                      (cudaStream_t)stream, what);
      };
      return a->residual_dtype == FERRUM_F32 ? go(float()) : go(T());
    });
  });
}

}  // extern "C"
