// Long causal convolution along the last axis of (batch, channels, length):
//   y[t] = sum_{s <= min(t, K-1)} k[s] x[t-s] + skip x[t]
//   dx[t] = sum_{s < K, t+s < L} k[s] dy[t+s] + skip dy[t]
//   dk[s] = sum_b sum_t dy[t] x[t-s],   dskip = dk[0]
// skip is added to k[0] when the filter is read, so it costs nothing.
//
// Through the FFT, a row of L real values is padded to 2M >= 2L and taken as
// the M-point complex sequence z[n] = x[2n] + i x[2n+1]. With Xe, Xo the
// transforms of the even and odd values (Xe = (Z[j] + conj Z[M-j]) / 2,
// i Xo = (Z[j] - conj Z[M-j]) / 2) and W = exp(-2 pi i j / M), the product of
// two such polynomials has the even part Xe Ke + W Xo Ko and the odd part
// Xe Ko + Xo Ke, so the convolution's transform is
//   Y[j] = alpha Z[j] + beta conj Z[M-j],
//   alpha = Ke + i Ko (1 - W) / 2,   beta = i Ko (1 + W) / 2,
// and its inverse holds (even, odd) outputs again. Rows are never paired, so
// nothing of one row (a NaN, a large value's rounding) reaches another.
// Correlation (dx, dk) takes the reversed filter: conj Ke and conj (W Ko).
//
// Up to M = 8192 one kernel takes a row through both transforms with one read
// and one write of it (the butterflies and exchanges of stockham.cuh, and one
// more exchange for Z[M-j]); longer rows go through the library's multi-pass
// transforms. Short rows take the defining sum.
// Measured, 8 x 1024 x 4096, bf16: 271 us, of which the filter's transform 20;
// two 4096-point transforms a row alone (no factor loads) 190. Exchanges in
// shared memory (62 % of its bandwidth), issue slots (51 %) and the waits for
// the factors bound it; HBM would take 23 us. With dx and dk 677 us.
#include <algorithm>

#include "../fft_kernels.cuh"
#include "seq_common.cuh"

namespace ferrum {
namespace seq {
namespace {

constexpr int kThreads = 256;

struct LongSizes {
  int64_t batch, channels, length, taps, blocks;  // blocks: thread blocks per row
};

template <class T>
__global__ void __launch_bounds__(kThreads)
direct_kernel(Rows<T> x, Rows<T> y, const float* __restrict__ k, const float* __restrict__ skip,
              LongSizes s, bool transposed, int64_t xs, int64_t ys) {
  const int64_t row = blockIdx.x / s.blocks;
  const int64_t t = (blockIdx.x % s.blocks) * kThreads + threadIdx.x;
  if (t >= s.length) return;
  const int64_t b = row / s.channels, d = row % s.channels;
  const T* xr = x.at(b, d);
  const float* kd = k + d * s.taps;
  const int64_t reach = transposed ? s.length - 1 - t : t;
  const int64_t n = reach < s.taps - 1 ? reach : s.taps - 1;
  float v = skip ? skip[d] * to_f(xr[t * xs]) : 0.f;
  for (int64_t i = 0; i <= n; ++i) v = fmaf(kd[i], to_f(xr[(transposed ? t + i : t - i) * xs]), v);
  y.at(b, d)[t * ys] = from_f<T>(v);
}

template <class T>
__global__ void __launch_bounds__(kThreads)
direct_dk_kernel(Rows<T> x, Rows<T> dy, float* __restrict__ dk, float* __restrict__ dskip,
                 LongSizes s, int64_t blocks, int64_t xs, int64_t gs) {
  const int64_t d = blockIdx.x / blocks;
  const int64_t i = (blockIdx.x % blocks) * kThreads + threadIdx.x;
  if (i >= s.taps) return;
  float v = 0.f;
  for (int64_t b = 0; b < s.batch; ++b) {
    float r = 0.f;
    const T *xr = x.at(b, d), *g = dy.at(b, d);
    for (int64_t t = i; t < s.length; ++t) r = fmaf(to_f(g[t * gs]), to_f(xr[(t - i) * xs]), r);
    v += r;
  }
  dk[d * s.taps + i] = v;
  if (dskip && i == 0) dskip[d] = v;
}

// One token: x goes into the history at its sequence's position, and the
// history up to there, reversed, meets the filter. One block per (b, d), each
// thread one value at a time: waits on loads bound it (8 x 1024 x 8192, bf16:
// 127 us, where history and filter once would take 26; 1 x 1024 x 1024 10 us, of
// which a launch is most).
template <class T>
__global__ void __launch_bounds__(kThreads)
long_step_kernel(Rows<T> x, Rows<T> y, Rows<T> hist, const int32_t* __restrict__ positions,
                 const float* __restrict__ k, const float* __restrict__ skip, LongSizes s) {
  __shared__ float sh[kThreads / 32];
  const int64_t b = blockIdx.x / s.channels, d = blockIdx.x % s.channels;
  const int64_t pos = positions[b];
  if (pos < 0 || pos >= s.length) {
    if (threadIdx.x == 0) y.at(b, 0)[d] = from_f<T>(0.f);
    return;
  }
  const T xv = x.at(b, 0)[d];
  T* h = hist.at(b, d);
  const float* kd = k + d * s.taps;
  if (threadIdx.x == 0) h[pos] = xv;
  float v = 0.f;
  for (int64_t i = 1 + threadIdx.x; i <= pos && i < s.taps; i += kThreads)
    v = fmaf(kd[i], to_f(h[pos - i]), v);
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    v = kd[0] * to_f(xv);
    for (int i = 0; i < kThreads / 32; ++i) v += sh[i];
    if (skip) v = fmaf(skip[d], to_f(xv), v);
    y.at(b, 0)[d] = from_f<T>(v);
  }
}

// ---------------------------------------------------------------- transforms
__device__ __forceinline__ float2 conj2(float2 a) { return make_float2(a.x, -a.y); }
// a * i
__device__ __forceinline__ float2 mul_i(float2 a) { return make_float2(-a.y, a.x); }
__device__ __forceinline__ float2 scale2(float2 a, float s) { return make_float2(a.x * s, a.y * s); }

// Spectra of the even and odd values from Z[j] and Z[M-j].
__device__ __forceinline__ void split_spectrum(float2 z, float2 zm, float2& e, float2& o) {
  e = make_float2(0.5f * (z.x + zm.x), 0.5f * (z.y - zm.y));
  o = make_float2(0.5f * (z.y + zm.y), 0.5f * (zm.x - z.x));
}

// alpha, beta of the filter with even and odd spectra ke, ko (`reversed`: of
// its time reversal), times `scale`.
__device__ __forceinline__ float4 filter_factors(float2 ke, float2 ko, float2 w, bool reversed,
                                                 float scale) {
  if (reversed) ke = conj2(ke), ko = conj2(c_mul(w, ko));
  const float2 iko = scale2(mul_i(ko), 0.5f * scale);
  const float2 b = c_mul(iko, w);
  const float2 a = c_add(scale2(ke, scale), c_sub(iko, b));
  const float2 beta = c_add(iko, b);
  return make_float4(a.x, a.y, beta.x, beta.y);
}

// Values 2q and 2q+1 of a row of n values, zeros past its end.
template <class T>
__device__ __forceinline__ float2 load_values(const T* p, int64_t q, int64_t n, bool vec) {
  const int64_t i = 2 * q;
  if (i + 1 < n) {
    if (vec) {
      if constexpr (std::is_same<T, float>::value) return *(const float2*)(p + i);
      if constexpr (std::is_same<T, __half>::value) return __half22float2(*(const __half2*)(p + i));
      if constexpr (std::is_same<T, __nv_bfloat16>::value)
        return __bfloat1622float2(*(const __nv_bfloat162*)(p + i));
    }
    return make_float2(to_f(p[i]), to_f(p[i + 1]));
  }
  return make_float2(i < n ? to_f(p[i]) : 0.f, 0.f);
}
template <class T>
__device__ __forceinline__ void store_values(T* p, int64_t q, int64_t n, float2 v, bool vec) {
  const int64_t i = 2 * q;
  if (i >= n) return;
  if (vec && i + 1 < n) {
    if constexpr (sizeof(T) == 4)
      *(float2*)(p + i) = make_float2(v.x, v.y);
    else
      *(uint32_t*)(p + i) = pack_pair<T>(v.x, v.y);
    return;
  }
  p[i] = from_f<T>(v.x);
  if (i + 1 < n) p[i + 1] = from_f<T>(v.y);
}

template <int LOGM>
struct LongCfg {
  static constexpr int LOGP = plan_log_p(LOGM);
  using G = Geom<LOGM, LOGP>;
  static constexpr int FPB = G::T >= 256 ? 1 : 256 / G::T;   // rows per block
  static constexpr int THREADS = FPB * G::T;
  static constexpr int RS = RegionStride<LOGM, LOGP, G::T >= 16 ? 1 : 16 / G::T>::value;
  static constexpr size_t BYTES = (size_t)FPB * RS * sizeof(float2);
  // Blocks an SM that the registers must allow for. The kernels wait on loads
  // (the factors, mostly), so warps count more than registers: rows_kernel at
  // 8 x 1024 x 4096 took 340, 328, 281 and 312 us with 2, 3, 4 and 5 blocks;
  // with 32 values a thread (M = 8192), 1362 us with 1 and 934 with 2. Shorter
  // rows alike: 2, 3, 4, 5 blocks at M = 128 193, 160, 144, 199 us, at 512 252, 215,
  // 197, 230, at 2048 287, 258, 240, 289 (33.5 M values in all). The
  // dkernel's sums take 32 or 64 registers more: 2 blocks up to M = 2048, 3 at
  // 4096 (forward + gradient 722 -> 689 us), 1 at 8192.
  static constexpr int ROW_BLOCKS = LOGM >= 13 ? 2 : 4;
  // rows_kernel's factors (16 bytes a bin, from the L2 cache) cost a quarter of
  // its time where each is loaded when it is needed (8 x 1024 x 4096 without
  // any loads: 211 us). What shared memory is left beside ROW_BLOCKS blocks
  // takes the first STAGED of a thread's P of them, copied while the first
  // transform runs: 281 -> 271 us, M = 8192 934 -> 840. (0, 5 and 8 staged at
  // M = 128 164, 144, 170 us; at 512 201, 197, 225; at 2048 246, 240, 264.)
  static constexpr int STAGED = LOGM >= 13 ? 10 : 5;
  static constexpr size_t ROW_BYTES = BYTES + sizeof(float4) * (size_t)(STAGED * THREADS);
  static constexpr int DK_BLOCKS = LOGM >= 13 ? 1 : (LOGM == 12 ? 3 : 2);
};

// Orders a row's threads: its warp, its warps, or the block.
template <int T, int FPB>
struct RowSync {
  int g;
  __device__ __forceinline__ void operator()() const {
    if constexpr (T <= 32)
      __syncwarp();
    else if constexpr (FPB == 1)
      __syncthreads();
    else
      SyncNamed{1 + g, T}();
  }
};

// v to shared memory in natural order, for reading Z[M-j].
template <int LOGM, class Sync>
__device__ __forceinline__ void put_spectrum(const float2 (&v)[1 << LongCfg<LOGM>::LOGP],
                                             float2* sm, int t, Sync sync) {
  using C = LongCfg<LOGM>;
  sync();   // the last exchange has been read
#pragma unroll
  for (int m = 0; m < C::G::P; ++m) sm[stage_read_addr<LOGM, C::LOGP>(t, m)] = v[m];
  sync();
}
template <int LOGM>
__device__ __forceinline__ float2 mirrored(const float2* sm, int t, int m) {
  using C = LongCfg<LOGM>;
  return sm[smem_pad<C::LOGP>(((1 << LOGM) - t - C::G::T * m) & ((1 << LOGM) - 1))];
}

// W_M^j from the two-level table.
template <int LOGM>
__device__ __forceinline__ float2 root(const float2* lo, const float2* hi, int j) {
  if constexpr (LOGM <= kFourStepLoBits)
    return __ldg(lo + j);
  else
    return four_step_twiddle(lo, hi, (uint32_t)j);
}

struct LongTables {
  const float2 *stage, *lo, *hi;
};

// A channel's alpha and beta (scaled by 1/M) to ab[d * M + j].
template <int LOGM>
__global__ void __launch_bounds__(LongCfg<LOGM>::THREADS, LongCfg<LOGM>::ROW_BLOCKS)
filter_kernel(const float* __restrict__ k, const float* __restrict__ skip, float4* __restrict__ ab,
              LongTables tw, LongSizes s, bool reversed) {
  using C = LongCfg<LOGM>;
  using G = typename C::G;
  extern __shared__ float2 sm_all[];
  const int g = threadIdx.x / G::T, t = threadIdx.x % G::T;
  const int64_t d = (int64_t)blockIdx.x * C::FPB + g;
  const bool ok = d < s.channels;
  float2* sm = sm_all + g * C::RS;
  const RowSync<G::T, C::FPB> sync{g};
  float2 v[G::P];
#pragma unroll
  for (int m = 0; m < G::P; ++m) {
    const int64_t q = t + G::T * m;
    v[m] = (ok && m < G::P / 2) ? load_values(k + d * s.taps, q, s.taps, false) : make_float2(0.f, 0.f);
    if (ok && q == 0 && skip) v[m].x += skip[d];
  }
  run_stages<LOGM, C::LOGP, 0>(v, sm, t, tw.stage, sync);
  put_spectrum<LOGM>(v, sm, t, sync);
  if (!ok) return;
  float4* out = ab + (d << LOGM);
#pragma unroll
  for (int m = 0; m < G::P; ++m) {
    float2 ke, ko;
    split_spectrum(v[m], mirrored<LOGM>(sm, t, m), ke, ko);
    out[t + G::T * m] = filter_factors(ke, ko, root<LOGM>(tw.lo, tw.hi, t + G::T * m), reversed,
                                       1.f / (float)G::N);
  }
}

// Rows through transform, product and inverse. Rows of a channel are
// neighbours, so its factors come from the L2 cache after the first.
template <class T, int LOGM>
__global__ void __launch_bounds__(LongCfg<LOGM>::THREADS, LongCfg<LOGM>::ROW_BLOCKS)
rows_kernel(Rows<T> x, Rows<T> y, const float4* __restrict__ ab, LongTables tw, LongSizes s,
            bool x_vec, bool y_vec) {
  using C = LongCfg<LOGM>;
  using G = typename C::G;
  extern __shared__ float2 sm_all[];
  const int g = threadIdx.x / G::T, t = threadIdx.x % G::T;
  const int64_t r = (int64_t)blockIdx.x * C::FPB + g;
  const bool ok = r < s.batch * s.channels;
  const int64_t d = ok ? r / s.batch : 0, b = ok ? r % s.batch : 0;
  float2* sm = sm_all + g * C::RS;
  const RowSync<G::T, C::FPB> sync{g};
  const T* xr = x.at(b, d);
  const float4* f = ab + (d << LOGM);
  float4* staged = (float4*)(sm_all + C::FPB * C::RS) + threadIdx.x;   // read back by this thread
#pragma unroll
  for (int m = 0; m < C::STAGED; ++m) cp_async<16>(staged + m * C::THREADS, f + t + G::T * m, 16);
  float2 v[G::P];
#pragma unroll
  for (int m = 0; m < G::P; ++m)
    v[m] = m < G::P / 2 ? load_values(xr, t + G::T * m, ok ? s.length : 0, x_vec)
                        : make_float2(0.f, 0.f);
  run_stages<LOGM, C::LOGP, 0>(v, sm, t, tw.stage, sync);
  put_spectrum<LOGM>(v, sm, t, sync);
  cp_async_wait();
#pragma unroll
  for (int m = 0; m < G::P; ++m) {
    const float4 c = m < C::STAGED ? staged[m * C::THREADS] : __ldg(f + t + G::T * m);
    const float2 u = c_add(c_mul(v[m], make_float2(c.x, c.y)),
                           c_mul(conj2(mirrored<LOGM>(sm, t, m)), make_float2(c.z, c.w)));
    v[m] = make_float2(u.y, u.x);     // swapped: the inverse by a forward transform
  }
  sync();
  run_stages<LOGM, C::LOGP, 0>(v, sm, t, tw.stage, sync);
  T* yr = y.at(b, d);
  if (!ok) return;
#pragma unroll
  for (int m = 0; m < G::P / 2; ++m)
    store_values(yr, t + G::T * m, s.length, make_float2(v[m].y, v[m].x), y_vec);
}

// dk of a channel over a share of the batch: the spectra of x and dy of each
// row, their correlation summed in registers, one inverse at the end.
template <class T, int LOGM>
__global__ void __launch_bounds__(LongCfg<LOGM>::THREADS, LongCfg<LOGM>::DK_BLOCKS)
dkernel_kernel(Rows<T> x, Rows<T> dy, float* __restrict__ dk, LongTables tw, LongSizes s,
               int64_t share, bool x_vec, bool dy_vec) {
  using C = LongCfg<LOGM>;
  using G = typename C::G;
  extern __shared__ float2 sm_all[];
  const int g = threadIdx.x / G::T, t = threadIdx.x % G::T;
  const int64_t chan_blocks = (s.channels + C::FPB - 1) / C::FPB;
  const int64_t d0 = (int64_t)(blockIdx.x % chan_blocks) * C::FPB + g, p = blockIdx.x / chan_blocks;
  const bool ok = d0 < s.channels;
  const int64_t d = ok ? d0 : 0;
  float2* sm = sm_all + g * C::RS;
  float2* sx = sm_all + (C::FPB + g) * C::RS;      // the spectrum of x
  const RowSync<G::T, C::FPB> sync{g};
  float2 acc[G::P];
#pragma unroll
  for (int m = 0; m < G::P; ++m) acc[m] = make_float2(0.f, 0.f);
  const int64_t b1 = (p + 1) * share < s.batch ? (p + 1) * share : s.batch;
  for (int64_t b = p * share; b < b1; ++b) {
    const T *xr = x.at(b, d), *gr = dy.at(b, d);
    float2 v[G::P];
#pragma unroll
    for (int m = 0; m < G::P; ++m)
      v[m] = m < G::P / 2 ? load_values(xr, t + G::T * m, s.length, x_vec) : make_float2(0.f, 0.f);
    run_stages<LOGM, C::LOGP, 0>(v, sm, t, tw.stage, sync);
    put_spectrum<LOGM>(v, sx, t, sync);
#pragma unroll
    for (int m = 0; m < G::P; ++m)
      v[m] = m < G::P / 2 ? load_values(gr, t + G::T * m, s.length, dy_vec) : make_float2(0.f, 0.f);
    run_stages<LOGM, C::LOGP, 0>(v, sm, t, tw.stage, sync);
    put_spectrum<LOGM>(v, sm, t, sync);
#pragma unroll
    for (int m = 0; m < G::P; ++m) {
      float2 xe, xo, ae, ao;
      split_spectrum(sx[stage_read_addr<LOGM, C::LOGP>(t, m)], mirrored<LOGM>(sx, t, m), xe, xo);
      split_spectrum(v[m], mirrored<LOGM>(sm, t, m), ae, ao);
      // even part: conj(xe) ae + conj(xo) ao; odd: conj(xe) ao + conj(W xo) ae
      const float2 w = root<LOGM>(tw.lo, tw.hi, t + G::T * m);
      xe = conj2(xe), xo = conj2(xo);
      const float2 e = c_add(c_mul(xe, ae), c_mul(xo, ao));
      const float2 o = c_add(c_mul(xe, ao), c_mul(c_mul(xo, conj2(w)), ae));
      acc[m] = c_add(acc[m], make_float2(e.x - o.y, e.y + o.x));
    }
    sync();
  }
  float2 v[G::P];
#pragma unroll
  for (int m = 0; m < G::P; ++m) v[m] = make_float2(acc[m].y, acc[m].x);
  run_stages<LOGM, C::LOGP, 0>(v, sm, t, tw.stage, sync);
  if (!ok) return;
  const float scale = 1.f / (float)G::N;
  float* out = dk + (p * s.channels + d) * s.taps;
#pragma unroll
  for (int m = 0; m < G::P / 2; ++m)
    store_values(out, t + G::T * m, s.taps, make_float2(v[m].y * scale, v[m].x * scale), false);
}

__global__ void first_column_kernel(const float* __restrict__ a, float* __restrict__ out, int64_t n,
                                    int64_t stride) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i < n) out[i] = a[i * stride];
}

// Rows of any step between contiguous and strided form: 32 x 32 tiles of
// (channel, step) through shared memory.
template <class T>
__global__ void restride_kernel(Rows<T> src, int64_t src_step, Rows<T> dst, int64_t dst_step,
                                int64_t channels, int64_t length, int64_t cb, int64_t tb) {
  __shared__ T tile[32][33];
  int64_t q = blockIdx.x;
  const int64_t t0 = q % tb * 32;
  q /= tb;
  const int64_t d0 = q % cb * 32, b = q / cb;
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  // lanes run along whichever axis of each side is closer together
  const bool st = src_step == 1, dt = dst_step == 1;
#pragma unroll
  for (int i = y; i < 32; i += 8) {
    const int64_t d = d0 + (st ? i : x), t = t0 + (st ? x : i);
    if (d < channels && t < length) tile[st ? i : x][st ? x : i] = src.at(b, d)[t * src_step];
  }
  __syncthreads();
#pragma unroll
  for (int i = y; i < 32; i += 8) {
    const int64_t d = d0 + (dt ? i : x), t = t0 + (dt ? x : i);
    if (d < channels && t < length) dst.at(b, d)[t * dst_step] = tile[dt ? i : x][dt ? x : i];
  }
}

// ---------------------------------------------------------------- multi-pass rows
// Row r of a chunk (r = (channel - d0) * batch + b) as M packed values.
template <class T>
__global__ void pack_kernel(Rows<T> x, float2* __restrict__ z, int log_m, LongSizes s, int64_t d0,
                            bool vec) {
  const int64_t m = (int64_t)1 << log_m;
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t r = i >> log_m, q = i & (m - 1);
  z[i] = load_values(x.at(r % s.batch, d0 + r / s.batch), q, s.length, vec);
}
template <class T>
__global__ void unpack_kernel(Rows<T> y, const float2* __restrict__ z, int log_m, LongSizes s,
                              int64_t d0, bool vec) {
  const int64_t half = (int64_t)1 << (log_m - 1);
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t r = i >> (log_m - 1), q = i & (half - 1);
  store_values(y.at(r % s.batch, d0 + r / s.batch), q, s.length, z[(r << log_m) + q], vec);
}
__global__ void pack_filter_kernel(const float* __restrict__ k, const float* __restrict__ skip,
                                   float2* __restrict__ z, int log_m, LongSizes s, int64_t d0) {
  const int64_t m = (int64_t)1 << log_m;
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t d = d0 + (i >> log_m), q = i & (m - 1);
  float2 v = load_values(k + d * s.taps, q, s.taps, false);
  if (q == 0 && skip) v.x += skip[d];
  z[i] = v;
}

// exp(-2 pi i j / M)
__device__ __forceinline__ float2 unit_root(int64_t j, int log_m) {
  float sn, cs;
  sincospif(-2.f * ((float)j / (float)((int64_t)1 << log_m)), &sn, &cs);
  return make_float2(cs, sn);
}

// z *= filter for a chunk's rows: one thread takes bins j and M-j.
__global__ void product_kernel(float2* __restrict__ z, const float2* __restrict__ k, int log_m,
                               LongSizes s, bool reversed) {
  const int64_t m = (int64_t)1 << log_m, half = m / 2;
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t r = i >> (log_m - 1);
  int64_t j = i & (half - 1);
  const float2* kr = k + ((r / s.batch) << log_m);
  float2* zr = z + (r << log_m);
  for (int pass = 0; pass < (j == 0 ? 2 : 1); ++pass) {
    const int64_t ja = pass ? half : j, jb = (m - ja) & (m - 1);
    const float2 za = zr[ja], zb = zr[jb];
    float2 ke, ko;
    split_spectrum(kr[ja], kr[jb], ke, ko);
    const float2 w = unit_root(ja, log_m);
    const float4 fa = filter_factors(ke, ko, w, reversed, 1.f);
    zr[ja] = c_add(c_mul(za, make_float2(fa.x, fa.y)), c_mul(conj2(zb), make_float2(fa.z, fa.w)));
    if (ja != jb) {
      const float4 fb = filter_factors(conj2(ke), conj2(ko), conj2(w), reversed, 1.f);
      zr[jb] = c_add(c_mul(zb, make_float2(fb.x, fb.y)), c_mul(conj2(za), make_float2(fb.z, fb.w)));
    }
  }
}

// Correlation spectra summed over the batch: out (channel, M) from x and dy.
__global__ void correlate_kernel(const float2* __restrict__ zx, const float2* __restrict__ zg,
                                 float2* __restrict__ out, int log_m, LongSizes s) {
  const int64_t m = (int64_t)1 << log_m;
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t d = i >> log_m, j = i & (m - 1), jm = (m - j) & (m - 1);
  const float2 w = conj2(unit_root(j, log_m));
  float2 acc = make_float2(0.f, 0.f);
  for (int64_t b = 0; b < s.batch; ++b) {
    const int64_t r = (d * s.batch + b) << log_m;
    float2 xe, xo, ae, ao;
    split_spectrum(zx[r + j], zx[r + jm], xe, xo);
    split_spectrum(zg[r + j], zg[r + jm], ae, ao);
    xe = conj2(xe), xo = conj2(xo);
    const float2 e = c_add(c_mul(xe, ae), c_mul(xo, ao));
    const float2 o = c_add(c_mul(xe, ao), c_mul(c_mul(xo, w), ae));
    acc = c_add(acc, make_float2(e.x - o.y, e.y + o.x));
  }
  out[i] = acc;
}
__global__ void unpack_filter_kernel(float* __restrict__ dk, const float2* __restrict__ z, int log_m,
                                     LongSizes s, int64_t d0) {
  const int64_t half = (int64_t)1 << (log_m - 1);
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t c = i >> (log_m - 1), q = i & (half - 1);
  store_values(dk + (d0 + c) * s.taps, q, s.taps, z[(c << log_m) + q], false);
}

ferrum_status check_long(const ferrum_device* dev, const ferrum_long_conv_args* a, const char* what,
                         bool bwd, bool step) {
  if (ferrum_status s = check_args(dev, a, what)) return s;
  if (a->length > FERRUM_LONG_CONV_MAX_LENGTH)
    return invalid(what, "length must be at most 2^25, got " + std::to_string(a->length));
  const bool none = a->batch == 0 || a->channels == 0, empty = none || a->length == 0;
  if (a->length > 0 && (a->kernel_length < 1 || a->kernel_length > a->length))
    return invalid(what, "kernel_length must be in [1, length], got " +
                             std::to_string(a->kernel_length));
  if (step && !none && a->length == 0) return invalid(what, "the history is empty");
  if (bounded_product({a->batch, a->channels, a->length}) < 0)
    return invalid(what, "batch * channels * length is too large");
  const size_t e = dtype_size(a->dtype);
  if (ferrum_status s = check_ptr(a->kernel, 4, empty, what, "kernel")) return s;
  if (ferrum_status s = check_ptr(a->skip, 4, true, what, "skip")) return s;
  if (ferrum_status s = check_ptr(a->x.ptr, e, empty, what, "x")) return s;
  if (step) {
    if (ferrum_status s = check_ptr(a->history.ptr, e, empty, what, "history")) return s;
    if (ferrum_status s = check_ptr(a->positions, 4, empty, what, "positions")) return s;
  }
  const int64_t out_step = bwd ? a->dx_step : a->y_step;
  if (!step && a->length > 1 && out_step == 0) return invalid(what, "the output's step is 0");
  if (!bwd) return check_ptr(a->y.ptr, e, empty, what, "y");
  if (ferrum_status s = check_ptr(a->dy.ptr, e, empty, what, "dy")) return s;
  if (ferrum_status s = check_ptr(a->dx.ptr, e, empty, what, "dx")) return s;
  if (ferrum_status s = check_ptr(a->dkernel, 4, a->channels == 0 || a->length == 0, what, "dkernel"))
    return s;
  return check_ptr(a->dskip, 4, true, what, "dskip");
}

LongSizes long_sizes(const ferrum_long_conv_args* a) {
  return LongSizes{(int64_t)a->batch, (int64_t)a->channels, (int64_t)a->length,
                   (int64_t)a->kernel_length, ceil_div((int64_t)a->length, kThreads)};
}


constexpr int kMaxFusedLog = 13;   // rows of up to 2^13 values in one kernel
// Rows up to here take the defining sum (us, forward: 1 x 64 rows of 64 values
// 10 against 18 through the FFT, 8 x 1024 rows 25 against 21, of 128 values 43
// against 21).
constexpr int64_t kDirectLength = 64;
constexpr int64_t kChunkBytes = (int64_t)1 << 30;   // spectra of the multi-pass path held at once

int log_rows(int64_t length) {     // log2 of M >= length
  int l = 7;
  while (((int64_t)1 << l) < length) ++l;
  return l;
}

template <class F>
ferrum_status with_log(int log_m, F f) {
  switch (log_m) {
    case 7: return f(std::integral_constant<int, 7>());
    case 8: return f(std::integral_constant<int, 8>());
    case 9: return f(std::integral_constant<int, 9>());
    case 10: return f(std::integral_constant<int, 10>());
    case 11: return f(std::integral_constant<int, 11>());
    case 12: return f(std::integral_constant<int, 12>());
    default: return f(std::integral_constant<int, 13>());
  }
}

// A row argument as the kernels take it: as it is where its step is 1, else
// through a contiguous copy in the workspace.
template <class T>
class Staged {
 public:
  Staged(ferrum_device* dev, const ferrum_rows& r, int64_t step, const LongSizes& s, bool in,
         cudaStream_t st)
      : user_(rows_of<T>(r)), step_(step), s_(s), st_(st),
        buf_(dev, step == 1 ? 0 : sizeof(T) * (size_t)(s.batch * s.channels * stride(s)), st) {
    rows_ = user_;
    if (step == 1) return;
    rows_ = Rows<T>{buf_.template as<T>(), s.channels * stride(s), stride(s)};
    if (in && buf_.status() == cudaSuccess) copy(user_, step_, rows_, 1);
  }
  cudaError_t status() const { return buf_.status(); }
  const Rows<T>& rows() const { return rows_; }
  // whether two values can be moved at once
  bool vec() const {
    return aligned(rows_.p, 2 * sizeof(T)) && rows_.sb % 2 == 0 && rows_.st % 2 == 0;
  }
  void finish() {   // an output's rows to the caller's array
    if (step_ != 1) copy(rows_, 1, user_, step_);
  }

 private:
  static int64_t stride(const LongSizes& s) { return (s.length + 7) / 8 * 8; }
  void copy(const Rows<T>& a, int64_t as, const Rows<T>& b, int64_t bs) {
    const int64_t cb = ceil_div(s_.channels, 32), tb = ceil_div(s_.length, 32);
    restride_kernel<T><<<(unsigned)(s_.batch * cb * tb), 256, 0, st_>>>(a, as, b, bs, s_.channels,
                                                                       s_.length, cb, tb);
  }
  Rows<T> user_, rows_;
  int64_t step_;
  LongSizes s_;
  cudaStream_t st_;
  PoolBuffer buf_;
};

template <class K>
ferrum_status allow_smem(K kernel, size_t bytes, std::atomic<uint64_t>& done, const char* what) {
  cudaError_t e = launch_detail::ensure_smem(kernel, bytes, done);
  return e == cudaSuccess ? FERRUM_OK : cuda_error(e, what);
}

// y (or, reversed, dx) of every row in one kernel.
template <class T>
ferrum_status fused_rows(ferrum_device* dev, const Staged<T>& x, const Staged<T>& y,
                         const float* k, const float* skip, const LongSizes& s, bool reversed,
                         cudaStream_t st, const char* what) {
  const int log_m = log_rows(s.length);
  PoolBuffer ab(dev, sizeof(float4) * (size_t)(s.channels << log_m), st);
  if (ab.status() != cudaSuccess) return cuda_error(ab.status(), "workspace");
  const LongTables tw{stage_table(dev, log_m), tw4_lo_table(dev, log_m), tw4_hi_table(dev, log_m)};
  return with_log(log_m, [&](auto l) -> ferrum_status {
    constexpr int L = decltype(l)::value;
    using C = LongCfg<L>;
    static std::atomic<uint64_t> done_f{0}, done_r{0};
    if (ferrum_status r = allow_smem(filter_kernel<L>, C::BYTES, done_f, what)) return r;
    if (ferrum_status r = allow_smem(rows_kernel<T, L>, C::ROW_BYTES, done_r, what)) return r;
    launch_detail::clear_stale_error();
    filter_kernel<L><<<(unsigned)ceil_div(s.channels, C::FPB), C::THREADS, C::BYTES, st>>>(
        k, skip, ab.as<float4>(), tw, s, reversed);
    rows_kernel<T, L>
        <<<(unsigned)ceil_div(s.batch * s.channels, C::FPB), C::THREADS, C::ROW_BYTES, st>>>(
            x.rows(), y.rows(), ab.as<float4>(), tw, s, x.vec(), y.vec());
    return launched(what);
  });
}

template <class T>
ferrum_status fused_dkernel(ferrum_device* dev, const Staged<T>& x, const Staged<T>& dy, float* dk,
                            const LongSizes& s, cudaStream_t st, const char* what) {
  const int log_m = log_rows(s.length);
  const LongTables tw{stage_table(dev, log_m), tw4_lo_table(dev, log_m), tw4_hi_table(dev, log_m)};
  return with_log(log_m, [&](auto l) -> ferrum_status {
    constexpr int L = decltype(l)::value;
    using C = LongCfg<L>;
    static std::atomic<uint64_t> done{0};
    if (ferrum_status r = allow_smem(dkernel_kernel<T, L>, 2 * C::BYTES, done, what)) return r;
    // few channels: the batch is shared out too, and the shares added in order
    const int64_t cb = ceil_div(s.channels, C::FPB);
    int64_t parts = std::min(s.batch, std::max<int64_t>(1, 148 * 2 / cb));
    const int64_t share = parts > 0 ? ceil_div(s.batch, parts) : 1;
    parts = std::max<int64_t>(1, ceil_div(s.batch, share));
    PoolBuffer ws(dev, parts > 1 ? sizeof(float) * (size_t)(parts * s.channels * s.taps) : 0, st);
    if (ws.status() != cudaSuccess) return cuda_error(ws.status(), "workspace");
    launch_detail::clear_stale_error();
    dkernel_kernel<T, L><<<(unsigned)(cb * parts), C::THREADS, 2 * C::BYTES, st>>>(
        x.rows(), dy.rows(), parts > 1 ? ws.as<float>() : dk, tw, s, share, x.vec(), dy.vec());
    if (ferrum_status r = launched(what)) return r;
    if (parts == 1) return FERRUM_OK;
    cudaError_t e = launch_sum_rows(ws.as<float>(), parts, s.channels * s.taps,
                                    s.channels * s.taps, dk, nullptr, st);
    return e == cudaSuccess ? FERRUM_OK : cuda_error(e, what);
  });
}

// Rows too long for one kernel, some channels at a time: y from x (`x`, `y`),
// or dx from dy reversed, and dk from x and dy when `dk` is given.
template <class T>
ferrum_status long_rows(ferrum_device* dev, const Staged<T>& in, const Staged<T>& out,
                        const Staged<T>* x, const float* k, const float* skip, float* dk,
                        const LongSizes& s, bool reversed, cudaStream_t st, const char* what) {
  const int log_m = log_rows(s.length);
  const int64_t per = (s.batch * (dk ? 2 : 1) + 1) * (int64_t)sizeof(float2) << log_m;
  const int64_t chunk = std::min(s.channels, std::max<int64_t>(1, kChunkBytes / per));
  const int64_t rows = chunk * s.batch;
  const size_t ws_bytes = workspace_1d_bytes(log_m, std::max(rows, chunk));
  PoolBuffer zin(dev, sizeof(float2) * (size_t)(std::max(rows, chunk) << log_m), st);
  PoolBuffer zk(dev, sizeof(float2) * (size_t)(chunk << log_m), st);
  PoolBuffer zx(dev, dk ? sizeof(float2) * (size_t)(rows << log_m) + 8 : 0, st);
  PoolBuffer ws(dev, ws_bytes, st);
  for (const PoolBuffer* p : {&zin, &zk, &zx, &ws})
    if (p->status() != cudaSuccess) return cuda_error(p->status(), "workspace");
  auto fft = [&](float2* z, int64_t n, int dir) {
    return enqueue_1d(dev, z, z, log_m, n, dir, dir < 0, ws.as<float2>(), st);
  };
  auto grid = [&](int64_t n) { return (unsigned)ceil_div(n, 256); };
  for (int64_t d0 = 0; d0 < s.channels; d0 += chunk) {
    const int64_t n = std::min(chunk, s.channels - d0), r = n * s.batch;
    float2 *z = zin.as<float2>(), *kz = zk.as<float2>(), *xz = zx.as<float2>();
    launch_detail::clear_stale_error();
    if (r > 0) {
      pack_kernel<T><<<grid(r << log_m), 256, 0, st>>>(in.rows(), z, log_m, s, d0, in.vec());
      if (ferrum_status e = launched(what)) return e;
      if (ferrum_status e = fft(z, r, 1)) return e;
    }
    if (dk) {
      if (r > 0) {
        pack_kernel<T><<<grid(r << log_m), 256, 0, st>>>(x->rows(), xz, log_m, s, d0, x->vec());
        if (ferrum_status e = launched(what)) return e;
        if (ferrum_status e = fft(xz, r, 1)) return e;
      }
      correlate_kernel<<<grid(n << log_m), 256, 0, st>>>(xz, z, kz, log_m, s);
      if (ferrum_status e = launched(what)) return e;
      if (ferrum_status e = fft(kz, n, -1)) return e;
      unpack_filter_kernel<<<grid(n << (log_m - 1)), 256, 0, st>>>(dk, kz, log_m, s, d0);
      if (ferrum_status e = launched(what)) return e;
    }
    if (r == 0) continue;
    pack_filter_kernel<<<grid(n << log_m), 256, 0, st>>>(k, skip, kz, log_m, s, d0);
    if (ferrum_status e = launched(what)) return e;
    if (ferrum_status e = fft(kz, n, 1)) return e;
    product_kernel<<<grid(r << (log_m - 1)), 256, 0, st>>>(z, kz, log_m, s, reversed);
    if (ferrum_status e = launched(what)) return e;
    if (ferrum_status e = fft(z, r, -1)) return e;
    unpack_kernel<T><<<grid(r << (log_m - 1)), 256, 0, st>>>(out.rows(), z, log_m, s, d0, out.vec());
    if (ferrum_status e = launched(what)) return e;
  }
  return FERRUM_OK;
}

}  // namespace
}  // namespace seq
}  // namespace ferrum

using namespace ferrum;
using namespace ferrum::seq;

extern "C" {

ferrum_status ferrum_long_conv(ferrum_device* dev, const ferrum_long_conv_args* a, void* stream) {
  const char* what = "long_conv";
  return guarded(what, [&]() -> ferrum_status {
    if (ferrum_status s = check_long(dev, a, what, false, false)) return s;
    if (a->batch == 0 || a->channels == 0 || a->length == 0) return FERRUM_OK;
    cudaStream_t st = (cudaStream_t)stream;
    const LongSizes s = long_sizes(a);
    const int64_t blocks =
        s.batch * std::max(s.channels * s.blocks, ceil_div(s.channels, 32) * ceil_div(s.length, 32));
    if (blocks > 0x7fffffff) return invalid(what, "too many blocks for one launch");
    DeviceGuard guard(dev->ordinal);
    if (guard.status() != cudaSuccess) return cuda_error(guard.status(), "cudaSetDevice");
    return with_dtype(a->dtype, [&](auto tag) -> ferrum_status {
      using T = decltype(tag);
      launch_detail::clear_stale_error();
      if (s.length <= kDirectLength) {
        direct_kernel<T><<<(unsigned)(s.batch * s.channels * s.blocks), kThreads, 0, st>>>(
            rows_of<T>(a->x), rows_of<T>(a->y), a->kernel, a->skip, s, false, a->x_step, a->y_step);
        return launched(what);
      }
      Staged<T> x(dev, a->x, a->x_step, s, true, st), y(dev, a->y, a->y_step, s, false, st);
      if (x.status() != cudaSuccess) return cuda_error(x.status(), "workspace");
      if (y.status() != cudaSuccess) return cuda_error(y.status(), "workspace");
      ferrum_status r =
          log_rows(s.length) <= kMaxFusedLog
              ? fused_rows<T>(dev, x, y, a->kernel, a->skip, s, false, st, what)
              : long_rows<T>(dev, x, y, nullptr, a->kernel, a->skip, nullptr, s, false, st, what);
      if (r) return r;
      y.finish();
      return launched(what);
    });
  });
}

ferrum_status ferrum_long_conv_bwd(ferrum_device* dev, const ferrum_long_conv_args* a,
                                   void* stream) {
  const char* what = "long_conv_bwd";
  return guarded(what, [&]() -> ferrum_status {
    if (ferrum_status s = check_long(dev, a, what, true, false)) return s;
    if (a->channels == 0 || a->length == 0) return FERRUM_OK;
    cudaStream_t st = (cudaStream_t)stream;
    const LongSizes s = long_sizes(a);
    const int64_t blocks =
        s.batch * std::max(s.channels * s.blocks, ceil_div(s.channels, 32) * ceil_div(s.length, 32));
    const int64_t kb = ceil_div(s.taps, kThreads);
    if (blocks > 0x7fffffff || kb * s.channels > 0x7fffffff)
      return invalid(what, "too many blocks for one launch");
    DeviceGuard guard(dev->ordinal);
    if (guard.status() != cudaSuccess) return cuda_error(guard.status(), "cudaSetDevice");
    return with_dtype(a->dtype, [&](auto tag) -> ferrum_status {
      using T = decltype(tag);
      launch_detail::clear_stale_error();
      if (s.length <= kDirectLength || s.batch == 0) {
        if (blocks > 0)
          direct_kernel<T><<<(unsigned)(s.batch * s.channels * s.blocks), kThreads, 0, st>>>(
              rows_of<T>(a->dy), rows_of<T>(a->dx), a->kernel, a->skip, s, true, a->dy_step,
              a->dx_step);
        direct_dk_kernel<T><<<(unsigned)(kb * s.channels), kThreads, 0, st>>>(
            rows_of<T>(a->x), rows_of<T>(a->dy), a->dkernel, a->dskip, s, kb, a->x_step, a->dy_step);
        return launched(what);
      }
      Staged<T> x(dev, a->x, a->x_step, s, true, st), dy(dev, a->dy, a->dy_step, s, true, st);
      Staged<T> dx(dev, a->dx, a->dx_step, s, false, st);
      for (const Staged<T>* p : {&x, &dy, &dx})
        if (p->status() != cudaSuccess) return cuda_error(p->status(), "workspace");
      ferrum_status r;
      if (log_rows(s.length) <= kMaxFusedLog) {
        r = fused_rows<T>(dev, dy, dx, a->kernel, a->skip, s, true, st, what);
        if (!r) r = fused_dkernel<T>(dev, x, dy, a->dkernel, s, st, what);
      } else {
        r = long_rows<T>(dev, dy, dx, &x, a->kernel, a->skip, a->dkernel, s, true, st, what);
      }
      if (r) return r;
      dx.finish();
      if (a->dskip)
        first_column_kernel<<<(unsigned)ceil_div(s.channels, 256), 256, 0, st>>>(
            a->dkernel, a->dskip, s.channels, s.taps);
      return launched(what);
    });
  });
}

ferrum_status ferrum_long_conv_step(ferrum_device* dev, const ferrum_long_conv_args* a,
                                    void* stream) {
  const char* what = "long_conv_step";
  return guarded(what, [&]() -> ferrum_status {
    if (ferrum_status s = check_long(dev, a, what, false, true)) return s;
    if (a->batch == 0 || a->channels == 0) return FERRUM_OK;
    const LongSizes s = long_sizes(a);
    if (s.batch * s.channels > 0x7fffffff) return invalid(what, "too many blocks for one launch");
    DeviceGuard guard(dev->ordinal);
    if (guard.status() != cudaSuccess) return cuda_error(guard.status(), "cudaSetDevice");
    return with_dtype(a->dtype, [&](auto tag) {
      using T = decltype(tag);
      launch_detail::clear_stale_error();
      long_step_kernel<T><<<(unsigned)(s.batch * s.channels), kThreads, 0, (cudaStream_t)stream>>>(
          rows_of<T>(a->x), rows_of<T>(a->y), rows_of<T>(a->history), a->positions, a->kernel,
          a->skip, s);
      return launched(what);
    });
  });
}

}  // extern "C"
