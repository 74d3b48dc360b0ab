// Dropout from a counter-based generator, added onto a residual:
//   y = residual + (word(i) >= p 2^32 ? x / (1 - p) : 0)
// word(i) is word i % 4 of Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel
// random numbers: as easy as 1, 2, 3", SC 2011) of counter (i / 4, offset) and key
// seed. Element i's word depends on nothing else, so no mask is stored, the
// gradient draws the same words, and neither strides nor the launch change them.
// A dropped value is selected away, not multiplied: an infinity or NaN there
// leaves no trace.
//
// A thread takes one to four groups of 8 adjacent elements: 16-byte accesses, and the
// 20 words of the generator's key schedule computed once for its counters. Contiguous
// arrays are one row, whatever their shape. 16384 x 2048 bf16 onto float32: 51 us,
// 6.5 TB/s, the rate of a copy; the gradient 39 us, 5.2 TB/s, half of its issue
// slots the generator's.
#include <type_traits>

#include "seq_common.cuh"

namespace ferrum {
namespace seq {
namespace {

constexpr int kThreads = 256;
constexpr int kVec = 8, kRounds = 10;

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
struct Keys {
  uint32_t k0[kRounds], k1[kRounds];
  __device__ __forceinline__ explicit Keys(uint64_t seed) {
#pragma unroll
    for (int r = 0; r < kRounds; ++r)
      k0[r] = (uint32_t)seed + r * 0x9E3779B9u, k1[r] = (uint32_t)(seed >> 32) + r * 0xBB67AE85u;
  }
};
__device__ __forceinline__ Words philox(uint64_t counter, uint64_t offset, const Keys& key) {
  uint32_t c0 = (uint32_t)counter, c1 = (uint32_t)(counter >> 32);
  uint32_t c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ key.k0[r], c2 = (uint32_t)(p0 >> 32) ^ c3 ^ key.k1[r];
    c1 = (uint32_t)p1, c3 = (uint32_t)p0;
  }
  return {{c0, c1, c2, c3}};
}

__device__ __forceinline__ float drop(uint32_t word, float x, float res, const Draw& d) {
  return word >= d.least && !d.none ? fmaf(x, d.scale, res) : res;
}

// kVec values as they lie in memory.
template <class T>
struct Raw {
  uint4 q[kVec * sizeof(T) / 16];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)(kVec * sizeof(T) / 16); ++i) q[i] = ((const uint4*)p)[i];
  }
  __device__ __forceinline__ void get(float (&v)[kVec]) const {
    const T* e = (const T*)q;
#pragma unroll
    for (int i = 0; i < kVec; ++i) v[i] = to_f(e[i]);
  }
};

// A group of up to kVec elements, the first of index `first`.
template <class T, class R>
__device__ __forceinline__ void drop_singly(const T* x, const R* res, R* y, uint64_t first, int n,
                                            const Draw& d, const Keys& key) {
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

// y = res + dropout(x). FLAT: one row (rows = 1). VEC says that all rows can be
// accessed a group of kVec at a time, which also means that a group starts at a
// multiple of 8 elements.
template <class T, class R, bool VEC, bool FLAT, int kGroups>
__global__ void __launch_bounds__(kThreads)
dropout_kernel(const T* __restrict__ x, const R* __restrict__ res, R* __restrict__ y,
               int64_t x_stride, int64_t res_stride, int64_t y_stride, int64_t channels,
               int64_t per_row, int64_t groups, Draw d) {
  const int64_t g0 = (int64_t)blockIdx.x * (kThreads * kGroups) + threadIdx.x;
  struct At {
    int64_t row, col;
  };
  auto place = [&](int64_t g) -> At {
    if (FLAT) return {0, g * kVec};
    if (groups <= 0xffffffffll)
      return {(int64_t)((uint32_t)g / (uint32_t)per_row), (int64_t)((uint32_t)g % (uint32_t)per_row) * kVec};
    return {g / per_row, g % per_row * kVec};
  };
  if constexpr (VEC) {
    const int64_t last = g0 + (kGroups - 1) * kThreads;
    if (FLAT ? (last + 1) * kVec <= channels : last < groups) {
      // All loads first, as they lie; the words are drawn while they are under way.
      Raw<T> v[kGroups];
      Raw<R> o[kGroups];
#pragma unroll
      for (int k = 0; k < kGroups; ++k) {
        const At a = place(g0 + k * kThreads);
        v[k].load(x + a.row * x_stride + a.col);
        if (res) o[k].load(res + a.row * res_stride + a.col);
      }
      const Keys key(d.seed_ptr ? *d.seed_ptr : d.seed);
#pragma unroll
      for (int k = 0; k < kGroups; ++k) {
        const At a = place(g0 + k * kThreads);
        const uint64_t counter = (uint64_t)(a.row * channels + a.col) / 4;
        const Words w0 = philox(counter, d.offset, key), w1 = philox(counter + 1, d.offset, key);
        float in[kVec], out[kVec];
        v[k].get(in);
        if (res) {
          o[k].get(out);
        } else {
#pragma unroll
          for (int i = 0; i < kVec; ++i) out[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          out[i] = drop(w0.w[i], in[i], out[i], d);
          out[4 + i] = drop(w1.w[i], in[4 + i], out[4 + i], d);
        }
        store_vec<R, kVec>(y + a.row * y_stride + a.col, out);
      }
      return;
    }
  }
  // the last block, the end of a row, or rows that are not aligned
  const Keys key(d.seed_ptr ? *d.seed_ptr : d.seed);
#pragma unroll 1
  for (int k = 0; k < kGroups; ++k) {
    const int64_t g = g0 + k * kThreads;
    if (g >= groups) return;
    const At a = place(g);
    const int n = channels - a.col < kVec ? (int)(channels - a.col) : kVec;
    drop_singly(x + a.row * x_stride + a.col, res ? res + a.row * res_stride + a.col : nullptr,
                y + a.row * y_stride + a.col, (uint64_t)(a.row * channels + a.col), n, d, key);
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
  auto run = [&](auto v, auto f, auto k) -> ferrum_status {
    constexpr int kGroups = decltype(k)::value;
    const int64_t blocks = ceil_div(groups, kThreads * kGroups);
    if (blocks > 0x7fffffff) return invalid(what, "too many values for one launch");
    launch_detail::clear_stale_error();
    dropout_kernel<T, R, decltype(v)::value, decltype(f)::value, kGroups>
        <<<(unsigned)blocks, kThreads, 0, stream>>>((const T*)x, (const R*)res, (R*)y, xs, rs, ys,
                                                    channels, per_row, groups, d);
    return launched(what);
  };
  using Y = std::true_type;
  using N = std::false_type;
  using One = std::integral_constant<int, 1>;
  using Two = std::integral_constant<int, 2>;
  using Four = std::integral_constant<int, 4>;
  if (!vec) return flat ? run(N(), Y(), One()) : run(N(), N(), One());
  // Groups a thread (16384 x 2048, us, 1 / 2 / 4): bf16 onto float32 51.5 / 55.3 / 57.5,
  // onto bf16 51.5 / 41.2 / 49.5; the gradient from float32 45.4 / 45.3 / 39.0, from
  // bf16 43.5 / 37.3 / 37.1. More of them share a key schedule, but their loads want
  // registers that threads in flight would have.
  if (groups < 148 * 2 * kThreads * 4) return flat ? run(Y(), Y(), One()) : run(Y(), N(), One());
  if (res == nullptr) return flat ? run(Y(), Y(), Four()) : run(Y(), N(), Four());
  if (sizeof(R) == 4) return flat ? run(Y(), Y(), One()) : run(Y(), N(), One());
  return flat ? run(Y(), Y(), Two()) : run(Y(), N(), Two());
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
