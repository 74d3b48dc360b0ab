// Gated linear recurrence over (batch, length, channels), one state a channel
// (recurrence.cuh has a step's arithmetic).
//
// A warp owns 16 steps of a row of channels (64 forward in 16-bit types, else 32).
// It copies them to shared memory a turn ahead, turns them into factors and inputs
// in registers, and sums them up as one map h -> A h + Q, with A from the sum of
// the logarithms. The maps of a turn's warps (8 a block, 1 to 8 blocks of a
// cluster, joined over distributed shared memory) give each warp the state it
// starts from; it then walks its 16 steps and stores them. One pass over the
// data, no block waits for another that might not run.
//
// 8 x 2048 x 4096 bf16: 160 us forward, 3.3 TB/s of the 6.5 of a copy (57
// instructions a value, issue slots 71 % busy, special functions 52 %: five a value
// are 75 us); its gradient 293 us, 3.2 TB/s (114 instructions, 74 %). float32: 175 us,
// 6.1 TB/s, and 414, 4.5 TB/s. 1 x 8191 x 2048 bf16: 67 and 107 us, 10 and 16 turns
// one after the other. Where a warp has a decay above 1 (recurrence.cuh): 213 and 394,
// 209 and 462, 85 and 136. 128 registers and 14 to 15 warps an SM in both.
//
// Gradient, with G the gradient of the state:  G_t = dout_t + a_{t+1} G_{t+1}. The
// same backwards over time; the states come from those the forward saved in front
// of every 16 steps.
#include <algorithm>
#include <atomic>

#include "recurrence.cuh"

namespace ferrum {
namespace seq {
namespace {

constexpr int kSteps = FERRUM_RECURRENCE_SAVE_STEPS;    // of a warp and turn
constexpr int kMaxWarps = 8, kMaxCluster = 8;
constexpr int kStepThreads = 128;

template <class T>
struct RecArrays {
  Rows<T> x, ig, rg, out;
  Rows<T> dout, dx, dig, drg;
  const float* decay;
  const float* initial;
  float* final;
  const int32_t* lengths;
  float* saved;
  const float* dfinal;
  float* dinitial;
  float* part;                 // (batch * cluster, channels): sums of ddecay
  int64_t batch, length, channels, groups;
};

__device__ __forceinline__ int64_t valid_length(const int32_t* lengths, int64_t b, int64_t length) {
  if (lengths == nullptr) return length;
  const int64_t n = lengths[b];
  return n < 0 ? 0 : (n > length ? length : n);
}

__device__ __forceinline__ void cp_async_wait_older() { asm volatile("cp.async.wait_group 1;" ::: "memory"); }

__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() { cluster_arrive(), cluster_wait(); }
// The block's barrier for warps that come to it from different places of the code (as
// __syncthreads() is not meant for).
__device__ __forceinline__ void block_sync() { asm volatile("bar.sync 0;" ::: "memory"); }
// Stores to this CTA's shared variable in CTA `rank` of the cluster, which has started (the
// kernels arrive at the cluster's barrier first thing and wait there in front of their
// first turn, behind its copies).
__device__ __forceinline__ void store_at_rank(float2* p, uint32_t rank, float2 v) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(a)
               : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(a), "f"(v.x), "f"(v.y) : "memory");
}

// How the rows of a call lie: at multiples of 16 bytes, of 4 bytes with an even
// number of channels (16-bit types), or of an element (8 x 2048 x 4095: 226 us where
// 4096 channels take 160).
enum Lie { kWhole, kPaired, kSingle };

// A warp's rows of one array in shared memory: 16 steps of 32 * VL channels. Where
// rows do not begin at multiples of 16 bytes, a row's copy begins at the 16-byte
// unit that holds its first value, so up to 14 bytes in front of it come along, from
// the same unit; behind its last value nothing is read.
template <class T, int VL, int LIE>
struct Stage {
  static constexpr int kRow = 32 * VL * (int)sizeof(T), kPitch = kRow + (LIE == kWhole ? 0 : 16);
  static constexpr int kUnits = kPitch / 16, kBytes = kSteps * kPitch;
  // Steps [0, n) from `p` on, `st` values apart, `channels` of them.
  static __device__ __forceinline__ void fill(uint8_t* s, const T* p, int64_t st, int n, int channels,
                                              int lane) {
    if constexpr (LIE == kWhole) {
#pragma unroll
      for (int i = 0; i < kSteps * kUnits / 32; ++i) {
        const int e = i * 32 + lane, step = e / kUnits, unit = e % kUnits;
        const uint8_t* row = (const uint8_t*)(p + (step < n ? step : 0) * st);
        const int left = channels * (int)sizeof(T) - unit * 16;
        const int bytes = step >= n || left <= 0 ? 0 : (left < 16 ? left : 16);
        cp_async<16>(s + step * kPitch + unit * 16, row + (bytes ? unit * 16 : 0), bytes);
      }
    } else {
#pragma unroll
      for (int i = 0; i < (kSteps * kUnits + 31) / 32; ++i) {
        const int e = i * 32 + lane, step = e / kUnits, unit = e % kUnits;
        if (step >= n) break;
        const uint8_t* row = (const uint8_t*)(p + step * st);
        const int in_front = (int)((uintptr_t)row & 15);
        const int left = in_front + channels * (int)sizeof(T) - unit * 16;
        const int bytes = left < 0 ? 0 : (left < 16 ? left : 16);
        cp_async<16>(s + step * kPitch + unit * 16, row - in_front + (bytes ? unit * 16 : 0), bytes);
      }
    }
  }
  // Channels 2 * lane and the next one, else lane and lane + 32.
  static constexpr bool kPairs = LIE != kSingle && VL == 2;
  static __device__ __forceinline__ int channel(int lane, int e) {
    return kPairs ? 2 * lane + e : lane + 32 * e;
  }
  static __device__ __forceinline__ void load(const uint8_t* s, const T* p, int64_t st, int step, int lane,
                                              float (&v)[VL]) {
    const uint8_t* row = s + step * kPitch;
    // (the low bits of the row's address)
    if constexpr (LIE != kWhole)
      row += ((uint32_t)(uintptr_t)p + (uint32_t)step * (uint32_t)st * (uint32_t)sizeof(T)) & 15;
    if constexpr (kPairs) {
      load_vec<T, 2>((const T*)row + 2 * lane, v);
    } else {
#pragma unroll
      for (int e = 0; e < VL; ++e) v[e] = to_f(((const T*)row)[lane + 32 * e]);
    }
  }
  static __device__ __forceinline__ void store(T* row, int lane, int channels, const float (&v)[VL]) {
    if constexpr (kPairs) {
      if (2 * lane < channels) store_vec<T, 2>(row + 2 * lane, v);   // (channels is even)
    } else {
#pragma unroll
      for (int e = 0; e < VL; ++e)
        if (lane + 32 * e < channels) row[lane + 32 * e] = from_f<T>(v[e]);
    }
  }
};

// Maps of a turn's warps, and of its blocks, by parity of the turn: a warp is never
// two turns ahead of another.
template <int VL>
struct Exchange {
  float2 warp[2][kMaxWarps][32 * VL];            // factor's code, Q
  // (only clusters of several blocks have what follows)
  float log_a[kMaxWarps][32 * VL];
  float2 block[2][kMaxCluster][32 * VL];
  static constexpr size_t kAlone = sizeof(float2) * 2 * kMaxWarps * 32 * VL;
};

// The state in front of this warp's part of the turn, in the order that `first`
// and `dir` give (0 and 1 forwards, the last and -1 backwards); `carry` moves on to
// the state behind the turn.
template <int VL>
__device__ __forceinline__ void exchange(Exchange<VL>& x, int parity, int warp, int warps, uint32_t rank,
                                         uint32_t size, bool back, int lane, const Factor (&a)[VL],
                                         const float (&log_a)[VL], const float (&q)[VL],
                                         float (&carry)[VL], float (&h)[VL]) {
#pragma unroll
  for (int e = 0; e < VL; ++e) {
    x.warp[parity][warp][lane + 32 * e] = make_float2(a[e].code, q[e]);
    if (size > 1) x.log_a[warp][lane + 32 * e] = log_a[e];
  }
  block_sync();
  const int at = back ? warps - 1 - warp : warp;         // place in the walk
  float start[VL];
#pragma unroll
  for (int e = 0; e < VL; ++e) start[e] = carry[e];
  if (size > 1) {
    if (warp < VL) {          // warp e sums up the block for its 32 channels
      const int c = lane + 32 * warp;
      float sum = 0.f, q2 = 0.f;
      for (int i = 0; i < warps; ++i) {
        const int w = back ? warps - 1 - i : i;
        const float2 m = x.warp[parity][w][c];
        sum += x.log_a[w][c];
        q2 = Factor{m.x}.step(q2, m.y);
      }
      if (isnan(q2)) {
        q2 = 0.f;
#pragma unroll 1
        for (int i = 0; i < warps; ++i) {
          const float2 m = x.warp[parity][back ? warps - 1 - i : i][c];
          q2 = Factor{m.x}.step<true>(q2, m.y);
        }
      }
      const float2 m = make_float2(factor_of(sum).code, q2);
      for (uint32_t r = 0; r < size; ++r) store_at_rank(&x.block[parity][rank][c], r, m);
    }
    cluster_sync();
#pragma unroll
    for (int e = 0; e < VL; ++e) {
      for (uint32_t i = 0; i < size; ++i) {
        const uint32_t r = back ? size - 1 - i : i;
        if (r == rank) h[e] = carry[e];
        const float2 m = x.block[parity][r][lane + 32 * e];
        carry[e] = Factor{m.x}.step(carry[e], m.y);
      }
      for (int i = 0; i < at; ++i) {
        const float2 m = x.warp[parity][back ? warps - 1 - i : i][lane + 32 * e];
        h[e] = Factor{m.x}.step(h[e], m.y);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < VL; ++e) {
      for (int i = 0; i < warps; ++i) {
        if (i == at) h[e] = carry[e];
        const float2 m = x.warp[parity][back ? warps - 1 - i : i][lane + 32 * e];
        carry[e] = Factor{m.x}.step(carry[e], m.y);
      }
    }
  }
  // Walks that keep infinities cost more: only where these ended in NaN.
#pragma unroll
  for (int e = 0; e < VL; ++e) {
    if (!isnan(carry[e]) && !isnan(h[e])) continue;
    carry[e] = start[e];
#pragma unroll 1
    for (int i = 0; i < (int)(size > 1 ? size : warps); ++i) {
      const int r = back ? (int)(size > 1 ? size : warps) - 1 - i : i;
      if (size > 1 ? r == (int)rank : i == at) h[e] = carry[e];
      const float2 m = size > 1 ? x.block[parity][r][lane + 32 * e] : x.warp[parity][r][lane + 32 * e];
      carry[e] = Factor{m.x}.step<true>(carry[e], m.y);
    }
#pragma unroll 1
    for (int i = 0; size > 1 && i < at; ++i) {
      const float2 m = x.warp[parity][back ? warps - 1 - i : i][lane + 32 * e];
      h[e] = Factor{m.x}.step<true>(h[e], m.y);
    }
  }
}

template <class T, int VL, int LIE>
__global__ void __launch_bounds__(32 * kMaxWarps, 2) recurrence_fwd_kernel(RecArrays<T> p) {
  using S = Stage<T, VL, LIE>;
  extern __shared__ __align__(16) uint8_t raw[];
  Exchange<VL>& ex = *(Exchange<VL>*)raw;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps = blockDim.x / 32;
  const uint32_t rank = cluster_rank(), size = cluster_size();
  if (size > 1) cluster_arrive();     // waited for in front of the first store to another block
  uint8_t* stage = raw + (size > 1 ? sizeof(Exchange<VL>) : Exchange<VL>::kAlone) + warp * 6 * S::kBytes;
  const int64_t part = blockIdx.x / size, b = part / p.groups, d0 = part % p.groups * 32 * VL;
  const int channels = p.channels - d0 < 32 * VL ? (int)(p.channels - d0) : 32 * VL;
  const int64_t len = valid_length(p.lengths, b, p.length);
  const int64_t chunk = (int64_t)size * warps * kSteps, turns = (p.length + chunk - 1) / chunk;
  const int64_t saves = (p.length + kSteps - 1) / kSteps;
  int64_t t0 = ((int64_t)rank * warps + warp) * kSteps;
  float decay[VL], carry[VL];
#pragma unroll
  for (int e = 0; e < VL; ++e) {
    const int c = S::channel(lane, e);
    decay[e] = c < channels ? checked_decay(p.decay[d0 + c]) : 0.f;
    carry[e] = c < channels && p.initial ? p.initial[b * p.channels + d0 + c] : 0.f;
  }
  bool mild = true;
#pragma unroll
  for (int e = 0; e < VL; ++e) mild = mild && decay[e] >= 0.f && decay[e] <= kShortDecay;
  mild = __all_sync(0xffffffffu, mild);
  auto valid = [&](int64_t t) {
    return (int)(len - t < 0 ? 0 : (len - t < kSteps ? len - t : kSteps));
  };
  auto fill = [&](int64_t t, int buf) {
    const int n = valid(t);
    if (n > 0) {
      uint8_t* s = stage + buf * 3 * S::kBytes;
      S::fill(s, p.x.at(b, t) + d0, p.x.st, n, channels, lane);
      S::fill(s + S::kBytes, p.ig.at(b, t) + d0, p.ig.st, n, channels, lane);
      S::fill(s + 2 * S::kBytes, p.rg.at(b, t) + d0, p.rg.st, n, channels, lane);
    }
    cp_async_commit();
  };
  fill(t0, 0);
  if (size > 1) cluster_wait();
  for (int64_t turn = 0; turn < turns; ++turn, t0 += chunk) {
    const int parity = (int)(turn & 1), n = valid(t0);
    __syncwarp();
    if (turn + 1 < turns)
      fill(t0 + chunk, parity ^ 1);
    else
      cp_async_commit();
    cp_async_wait_older();
    __syncwarp();
    const uint8_t* s = stage + parity * 3 * S::kBytes;
    const T *px = p.x.at(b, t0) + d0, *pi = p.ig.at(b, t0) + d0, *pr = p.rg.at(b, t0) + d0;
    // SHORT: all steps inside the sequence, all decays in expm1_short's range
    auto walk = [&](auto is_short) {
      constexpr bool SHORT = decltype(is_short)::value;
      Factor a[kSteps][VL], all[VL];
      float in[kSteps][VL], sum[VL], q[VL], h[VL];
#pragma unroll
      for (int e = 0; e < VL; ++e) sum[e] = q[e] = 0.f;
#pragma unroll
      for (int j = 0; j < kSteps; ++j) {
        float x[VL], ig[VL], rg[VL];
        S::load(s, px, p.x.st, j, lane, x);
        S::load(s + S::kBytes, pi, p.ig.st, j, lane, ig);
        S::load(s + 2 * S::kBytes, pr, p.rg.st, j, lane, rg);
#pragma unroll
        for (int e = 0; e < VL; ++e) {
          const float r = sigmoid_f(rg[e]);
          float w;
          a[j][e] = step_factor<SHORT>(decay[e], r, w);
          in[j][e] = root_of(w) * (sigmoid_f(ig[e]) * x[e]);
          if (SHORT || j < n) sum[e] += r;
          if (!SHORT && j >= n) a[j][e].code = kKeep, in[j][e] = 0.f;
          q[e] = step_on<SHORT>(a[j][e], q[e], in[j][e]);
        }
      }
#pragma unroll
      for (int e = 0; e < VL; ++e) {
        if (isnan(q[e])) {              // (as in exchange())
          q[e] = 0.f;
#pragma unroll
          for (int j = 0; j < kSteps; ++j) q[e] = step_on<SHORT, true>(a[j][e], q[e], in[j][e]);
        }
      }
#pragma unroll
      for (int e = 0; e < VL; ++e) {
        sum[e] *= -decay[e];
        all[e] = factor_of(sum[e]);
      }
      exchange<VL>(ex, parity, warp, warps, rank, size, false, lane, all, sum, q, carry, h);
      if (t0 >= p.length) return;
      if (p.saved) {
#pragma unroll
        for (int e = 0; e < VL; ++e) {
          const int c = S::channel(lane, e);
          if (c < channels) p.saved[(b * saves + t0 / kSteps) * p.channels + d0 + c] = h[e];
        }
      }
      const int rows = p.length - t0 < kSteps ? (int)(p.length - t0) : kSteps;
      float start[VL];
#pragma unroll
      for (int e = 0; e < VL; ++e) start[e] = h[e];
      auto show = [&](auto any) {
        T* po = p.out.at(b, t0) + d0;
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
          if (!SHORT && j >= rows) break;
          float o[VL];
#pragma unroll
          for (int e = 0; e < VL; ++e) {
            h[e] = step_on<SHORT, any.value>(a[j][e], h[e], in[j][e]);
            o[e] = SHORT || j < n ? h[e] : 0.f;
          }
          S::store(po, lane, channels, o);
          po += p.out.st;
        }
      };
      show(std::false_type());
      bool lost = false;
#pragma unroll
      for (int e = 0; e < VL; ++e) lost = lost || isnan(h[e]), h[e] = start[e];
      if (lost) show(std::true_type());
    };
    // Behind the sequence's end the state stands still (8 sequences of 0 to 2048 steps x
    // 4096 bf16: 187 us where warps walk their padding, 123 where they do not; the
    // gradient 353 and 218).
    auto stand = [&] {
      Factor all[VL];
      float none[VL], h[VL];
#pragma unroll
      for (int e = 0; e < VL; ++e) all[e].code = kKeep, none[e] = 0.f;
      exchange<VL>(ex, parity, warp, warps, rank, size, false, lane, all, none, none, carry, h);
      if (t0 >= p.length) return;
      if (p.saved) {
#pragma unroll
        for (int e = 0; e < VL; ++e) {
          const int c = S::channel(lane, e);
          if (c < channels) p.saved[(b * saves + t0 / kSteps) * p.channels + d0 + c] = h[e];
        }
      }
      const int rows = p.length - t0 < kSteps ? (int)(p.length - t0) : kSteps;
      for (int j = 0; j < rows; ++j) S::store(p.out.at(b, t0 + j) + d0, lane, channels, none);
    };
    if (n == kSteps && mild)
      walk(std::true_type());
    else if (n > 0)
      walk(std::false_type());
    else
      stand();
  }
  if (p.final && warp == 0 && rank == 0) {
#pragma unroll
    for (int e = 0; e < VL; ++e) {
      const int c = S::channel(lane, e);
      if (c < channels) p.final[b * p.channels + d0 + c] = carry[e];
    }
  }
  if (size > 1) cluster_sync();       // no block ends while another may store to it
}

// (Blocks an SM by their shared memory: two of 8 warps, three of 4.)
template <class T, int LIE, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, WARPS == 8 ? 2 : 3) recurrence_bwd_kernel(RecArrays<T> p) {
  using S = Stage<T, 1, LIE>;
  extern __shared__ __align__(16) uint8_t raw[];
  Exchange<1>& ex = *(Exchange<1>*)raw;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps = blockDim.x / 32;
  const uint32_t rank = cluster_rank(), size = cluster_size();
  if (size > 1) cluster_arrive();     // waited for in front of the first store to another block
  uint8_t* stage = raw + (size > 1 ? sizeof(Exchange<1>) : Exchange<1>::kAlone) + warp * 8 * S::kBytes;
  const int64_t part = blockIdx.x / size, b = part / p.groups, d0 = part % p.groups * 32;
  const int channels = p.channels - d0 < 32 ? (int)(p.channels - d0) : 32;
  const bool mine = lane < channels;
  const int64_t len = valid_length(p.lengths, b, p.length), at = b * p.channels + d0 + lane;
  const int64_t chunk = (int64_t)size * warps * kSteps, turns = (p.length + chunk - 1) / chunk;
  const int64_t saves = (p.length + kSteps - 1) / kSteps;
  int64_t t0 = (turns - 1) * chunk + ((int64_t)rank * warps + warp) * kSteps;
  const float decay = mine ? checked_decay(p.decay[d0 + lane]) : 0.f;
  const bool mild = __all_sync(0xffffffffu, decay >= 0.f && decay <= kShortDecay);
  float carry[1] = {mine && p.dfinal ? p.dfinal[at] : 0.f}, total = 0.f;
  auto valid = [&](int64_t t) {
    return (int)(len - t < 0 ? 0 : (len - t < kSteps ? len - t : kSteps));
  };
  auto fill = [&](int64_t t, int buf) {
    const int n = valid(t);
    if (n > 0) {
      uint8_t* s = stage + buf * 4 * S::kBytes;
      S::fill(s, p.x.at(b, t) + d0, p.x.st, n, channels, lane);
      S::fill(s + S::kBytes, p.ig.at(b, t) + d0, p.ig.st, n, channels, lane);
      S::fill(s + 2 * S::kBytes, p.rg.at(b, t) + d0, p.rg.st, n, channels, lane);
      S::fill(s + 3 * S::kBytes, p.dout.at(b, t) + d0, p.dout.st, n, channels, lane);
    }
    cp_async_commit();
  };
  if (turns > 0) fill(t0, (int)(turns - 1) & 1);
  if (size > 1) cluster_wait();
  for (int64_t turn = turns - 1; turn >= 0; --turn, t0 -= chunk) {
    const int parity = (int)(turn & 1), n = valid(t0);
    __syncwarp();
    if (turn > 0)
      fill(t0 - chunk, parity ^ 1);
    else
      cp_async_commit();
    float h = n > 0 && mine ? p.saved[(b * saves + t0 / kSteps) * p.channels + d0 + lane] : 0.f;
    cp_async_wait_older();
    __syncwarp();
    const uint8_t* s = stage + parity * 4 * S::kBytes;
    const T *px = p.x.at(b, t0) + d0, *pi = p.ig.at(b, t0) + d0, *pr = p.rg.at(b, t0) + d0;
    const T* pg = p.dout.at(b, t0) + d0;
    // Every gradient of a step is its state's gradient g times a number that the
    // walk forwards computes: dx = g root i, dig = dx x (1 - i),
    // ddecay = -g r a (h - a / root i x), drg = ddecay decay (1 - r).
    auto walk = [&](auto is_short) {
      constexpr bool SHORT = decltype(is_short)::value;
      Factor a[kSteps];
      float fx[kSteps], fi[kSteps], fr[kSteps], fd[kSteps];
      float sum[1] = {0.f}, q[1] = {0.f}, later[1];
#pragma unroll
      for (int j = 0; j < kSteps; ++j) {
        float x[1], ig[1], rg[1], w;
        S::load(s, px, p.x.st, j, lane, x);
        S::load(s + S::kBytes, pi, p.ig.st, j, lane, ig);
        S::load(s + 2 * S::kBytes, pr, p.rg.st, j, lane, rg);
        const Gate i = gate_of(ig[0]), r = gate_of(rg[0]);
        a[j] = step_factor<SHORT>(decay, r.on, w);
        const float inv = inverse_root_of(w), factor = SHORT ? 1.f + a[j].code : a[j].value();
        fx[j] = w * inv * i.on;
        const float in = fx[j] * x[0];
        fi[j] = in * i.off;
        fd[j] = -r.on * factor * fmaf(-factor * inv, i.on * x[0], h);
        fr[j] = fd[j] * decay * r.off;
        if (SHORT || j < n) sum[0] += r.on;
        if (!SHORT && j >= n) a[j].code = kKeep;
        h = step_on<SHORT>(a[j], h, in);
      }
#pragma unroll
      for (int j = kSteps - 1; j >= 0; --j) {
        float g[1];
        S::load(s + 3 * S::kBytes, pg, p.dout.st, j, lane, g);
        q[0] = step_times<SHORT>(a[j], (SHORT || j < n ? g[0] : 0.f) + q[0]);
      }
      sum[0] *= -decay;
      const Factor all[1] = {factor_of(sum[0])};
      exchange<1>(ex, parity, warp, warps, rank, size, true, lane, all, sum, q, carry, later);
      if (t0 >= p.length) return;
      const int rows = p.length - t0 < kSteps ? (int)(p.length - t0) : kSteps;
      T* ox = p.dx.at(b, t0 + rows - 1) + d0 + lane;
      T* oi = p.dig.at(b, t0 + rows - 1) + d0 + lane;
      T* orr = p.drg.at(b, t0 + rows - 1) + d0 + lane;
#pragma unroll
      for (int j = kSteps - 1; j >= 0; --j) {
        if (!SHORT && j >= rows) continue;
        float g[1];
        S::load(s + 3 * S::kBytes, pg, p.dout.st, j, lane, g);
        const bool on = SHORT || j < n;
        g[0] += later[0];
        if (on) total = fmaf(g[0], fd[j], total), later[0] = step_times<SHORT>(a[j], g[0]);
        if (mine) {
          *ox = from_f<T>(on ? g[0] * fx[j] : 0.f);
          *oi = from_f<T>(on ? g[0] * fi[j] : 0.f);
          *orr = from_f<T>(on ? g[0] * fr[j] : 0.f);
        }
        ox -= p.dx.st, oi -= p.dig.st, orr -= p.drg.st;
      }
    };
    auto stand = [&] {
      const Factor all[1] = {{kKeep}};
      const float none[1] = {0.f};
      float later[1];
      exchange<1>(ex, parity, warp, warps, rank, size, true, lane, all, none, none, carry, later);
      if (t0 >= p.length || !mine) return;
      const int rows = p.length - t0 < kSteps ? (int)(p.length - t0) : kSteps;
      for (int j = 0; j < rows; ++j) {
        p.dx.at(b, t0 + j)[d0 + lane] = from_f<T>(0.f);
        p.dig.at(b, t0 + j)[d0 + lane] = from_f<T>(0.f);
        p.drg.at(b, t0 + j)[d0 + lane] = from_f<T>(0.f);
      }
    };
    if (n == kSteps && mild)
      walk(std::true_type());
    else if (n > 0)
      walk(std::false_type());
    else
      stand();
  }
  if (p.dinitial && mine && warp == 0 && rank == 0) p.dinitial[at] = carry[0];
  // the block's sum of ddecay, warp by warp
  __syncthreads();
  ex.warp[0][warp][lane].x = total;
  __syncthreads();
  if (warp == 0 && mine) {
    float v = 0.f;
    for (int w = 0; w < warps; ++w) v += ex.warp[0][w][lane].x;
    p.part[(b * size + rank) * p.channels + d0 + lane] = v;
  }
  if (size > 1) cluster_sync();
}

// One step of every sequence, VL channels a thread, each read before it is written.
template <class T, int VL>
__global__ void __launch_bounds__(kStepThreads) recurrence_step_kernel(RecArrays<T> p) {
  const uint32_t per = (uint32_t)(p.channels / VL);
  const int64_t i = (int64_t)blockIdx.x * kStepThreads + threadIdx.x;
  if (i >= p.batch * per) return;
  const int64_t b = i <= 0xffffffffll ? (uint32_t)i / per : i / per, d = (i - b * per) * VL;
  float x[VL], ig[VL], rg[VL], decay[VL], h[VL];
  load_vec<T, VL>(p.x.at(b, 0) + d, x);
  load_vec<T, VL>(p.ig.at(b, 0) + d, ig);
  load_vec<T, VL>(p.rg.at(b, 0) + d, rg);
  load_vec<float, VL>(p.decay + d, decay);
  load_vec<float, VL>(p.initial + b * p.channels + d, h);
#pragma unroll
  for (int e = 0; e < VL; ++e) {
    float w;
    const Factor a = factor_of(-checked_decay(decay[e]) * sigmoid_f(rg[e]), &w);
    h[e] = a.step<true>(h[e], root_of(w) * (sigmoid_f(ig[e]) * x[e]));
  }
  store_vec<T, VL>(p.out.at(b, 0) + d, h);
  store_vec<float, VL>(p.final + b * p.channels + d, h);
}

template <class T>
RecArrays<T> arrays_of(const ferrum_recurrence_args* a) {
  RecArrays<T> p;
  p.x = rows_of<T>(a->x), p.ig = rows_of<T>(a->input_gate), p.rg = rows_of<T>(a->recurrence_gate);
  p.out = rows_of<T>(a->out), p.dout = rows_of<T>(a->dout), p.dx = rows_of<T>(a->dx);
  p.dig = rows_of<T>(a->dinput_gate), p.drg = rows_of<T>(a->drecurrence_gate);
  p.decay = a->decay, p.initial = a->initial_state, p.final = a->final_state;
  p.lengths = a->lengths, p.saved = a->saved_states, p.dfinal = a->dfinal_state;
  p.dinitial = a->dinitial_state, p.part = nullptr, p.groups = 0;
  p.batch = (int64_t)a->batch, p.length = (int64_t)a->length, p.channels = (int64_t)a->channels;
  return p;
}

ferrum_status check_recurrence(const ferrum_device* dev, const ferrum_recurrence_args* a,
                               const char* what, bool bwd) {
  if (ferrum_status s = check_args(dev, a, what)) return s;
  if (bounded_product({a->batch, a->length, a->channels}) < 0 ||
      bounded_product({a->batch, a->channels}) < 0 || a->length > (size_t)kMaxElems)
    return invalid(what, "batch * length * channels is too large");
  const size_t e = dtype_size(a->dtype);
  const bool none = a->batch == 0 || a->channels == 0, empty = none || a->length == 0;
  struct {
    const void* p;
    size_t align;
    bool optional;
    const char* name;
  } const arrays[] = {
      {a->decay, 4, a->channels == 0, "decay"},
      {a->initial_state, 4, true, "initial_state"},
      {a->final_state, 4, true, "final_state"},
      {a->lengths, 4, true, "lengths"},
      {a->x.ptr, e, empty, "x"},
      {a->input_gate.ptr, e, empty, "input_gate"},
      {a->recurrence_gate.ptr, e, empty, "recurrence_gate"},
      {bwd ? a->dout.ptr : a->out.ptr, e, empty, bwd ? "dout" : "out"},
      {a->saved_states, 4, !bwd || empty, "saved_states"},
      {a->dx.ptr, e, !bwd || empty, "dx"},
      {a->dinput_gate.ptr, e, !bwd || empty, "dinput_gate"},
      {a->drecurrence_gate.ptr, e, !bwd || empty, "drecurrence_gate"},
      {a->dfinal_state, 4, true, "dfinal_state"},
      {a->ddecay, 4, !bwd || a->channels == 0, "ddecay"},
      {a->dinitial_state, 4, true, "dinitial_state"},
  };
  for (const auto& v : arrays)
    if (ferrum_status s = check_ptr(v.p, v.align, v.optional, what, v.name)) return s;
  return FERRUM_OK;
}

// Blocks of a cluster: more of them where there are few rows of channels, as long
// as each has steps to walk. With 1, 2, 4 and 8 blocks, us: 1 x 8191 x 2048 bf16
// forward 224, 156, 86, 66, gradient (twice the rows) 238, 159, 110, 114;
// 8 x 2048 x 4096 164, 209, 230, 311 and 310, 367, 395, 453.
int cluster_of(int64_t parts, int64_t length, int warps) {
  int c = 1;
  while (c < kMaxCluster && parts * c * 2 <= 148 * 2 && (int64_t)c * warps * kSteps < length) c *= 2;
  return c;
}

// Warps of a block, 16 steps each: no more than the steps need, nor than let two
// blocks share an SM's 228 KiB.
struct Shape {
  int cluster, warps;
  size_t smem;
};
template <class X>
Shape shape_of(int64_t parts, int64_t length, int most, size_t per_warp) {
  auto fit = [&](size_t fixed) {
    const int64_t room = (int64_t)((113 * 1024 - fixed) / per_warp);
    return (int)std::max<int64_t>(1, std::min<int64_t>({most, room, ceil_div(length, kSteps)}));
  };
  Shape s;
  s.warps = fit(X::kAlone);
  s.cluster = cluster_of(parts, length, s.warps);
  if (s.cluster > 1) s.warps = fit(sizeof(X));
  s.smem = (s.cluster > 1 ? sizeof(X) : X::kAlone) + s.warps * per_warp;
  return s;
}

bool rows_aligned(std::initializer_list<const ferrum_rows*> arrays, size_t e, int64_t bytes) {
  for (const ferrum_rows* r : arrays)
    if (!aligned(r->ptr, (size_t)bytes) || r->batch_stride * (int64_t)e % bytes != 0 ||
        r->row_stride * (int64_t)e % bytes != 0)
      return false;
  return true;
}

template <class K, class T>
ferrum_status launch(K kernel, std::atomic<uint64_t>& smem_done, const RecArrays<T>& p, const Shape& s,
                     cudaStream_t stream, const char* what) {
  const int64_t blocks = p.batch * p.groups * s.cluster;
  if (blocks > 0x7fffffff) return invalid(what, "too many blocks for one launch");
  cudaError_t e = launch_detail::ensure_smem(kernel, 113 * 1024, smem_done);
  if (e != cudaSuccess) return cuda_error(e, what);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)s.cluster, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks), cfg.blockDim = dim3(32 * s.warps);
  cfg.dynamicSmemBytes = s.smem, cfg.stream = stream, cfg.attrs = attr, cfg.numAttrs = 1;
  launch_detail::clear_stale_error();
  e = cudaLaunchKernelEx(&cfg, kernel, p);
  return e == cudaSuccess ? FERRUM_OK : cuda_error(e, what);
}

template <class T, int VL, int LIE>
ferrum_status run_fwd(RecArrays<T> p, cudaStream_t stream, const char* what) {
  static std::atomic<uint64_t> smem_done{0};
  p.groups = ceil_div(p.channels, 32 * VL);
  const Shape s = shape_of<Exchange<VL>>(p.batch * p.groups, p.length, kMaxWarps,
                                         6 * Stage<T, VL, LIE>::kBytes);
  return launch(recurrence_fwd_kernel<T, VL, LIE>, smem_done, p, s, stream, what);
}

template <class T, int LIE>
ferrum_status run_bwd(ferrum_device* dev, RecArrays<T> p, float* ddecay, cudaStream_t stream,
                      const char* what) {
  static std::atomic<uint64_t> smem_done{0};
  constexpr int kWarps = sizeof(T) == 4 ? 4 : 8;
  p.groups = ceil_div(p.channels, 32);
  const Shape s = shape_of<Exchange<1>>(p.batch * p.groups, p.length, kWarps,
                                        8 * Stage<T, 1, LIE>::kBytes);
  const int64_t sums = p.batch * s.cluster;
  PoolBuffer ws(dev, (size_t)(sums * p.channels) * 4 + 4, stream);
  if (ws.status() != cudaSuccess) return cuda_error(ws.status(), "workspace");
  p.part = ws.as<float>();
  if (p.batch > 0) {
    if (ferrum_status f = launch(recurrence_bwd_kernel<T, LIE, kWarps>, smem_done, p, s, stream, what))
      return f;
  }
  cudaError_t e = launch_sum_rows(p.part, sums, p.channels, p.channels, ddecay, nullptr, stream);
  return e == cudaSuccess ? FERRUM_OK : cuda_error(e, what);
}

}  // namespace
}  // namespace seq
}  // namespace ferrum

using namespace ferrum;
using namespace ferrum::seq;

extern "C" {

ferrum_status ferrum_gated_recurrence(ferrum_device* dev, const ferrum_recurrence_args* a,
                                      void* stream) {
  const char* what = "gated_recurrence";
  return guarded(what, [&]() -> ferrum_status {
    if (ferrum_status s = check_recurrence(dev, a, what, false)) return s;
    const int64_t n = (int64_t)a->batch * (int64_t)a->channels;
    if (n == 0) return FERRUM_OK;
    DeviceGuard guard(dev->ordinal);
    if (guard.status() != cudaSuccess) return cuda_error(guard.status(), "cudaSetDevice");
    return with_dtype(a->dtype, [&](auto tag) {
      using T = decltype(tag);
      constexpr int VL = sizeof(T) == 2 ? 2 : 1;
      cudaStream_t st = (cudaStream_t)stream;
      const RecArrays<T> p = arrays_of<T>(a);
      auto lie = [&](int64_t bytes) {
        return rows_aligned({&a->x, &a->input_gate, &a->recurrence_gate, &a->out}, sizeof(T), bytes);
      };
      const bool even = a->channels % VL == 0;
      if (even && lie(16)) return run_fwd<T, VL, kWhole>(p, st, what);
      if constexpr (VL == 2) {
        if (even && lie(4)) return run_fwd<T, VL, kPaired>(p, st, what);
      }
      return run_fwd<T, VL, kSingle>(p, st, what);
    });
  });
}

ferrum_status ferrum_gated_recurrence_bwd(ferrum_device* dev, const ferrum_recurrence_args* a,
                                          void* stream) {
  const char* what = "gated_recurrence_bwd";
  return guarded(what, [&]() -> ferrum_status {
    if (ferrum_status s = check_recurrence(dev, a, what, true)) return s;
    if (a->channels == 0) return FERRUM_OK;
    cudaStream_t st = (cudaStream_t)stream;
    DeviceGuard guard(dev->ordinal);
    if (guard.status() != cudaSuccess) return cuda_error(guard.status(), "cudaSetDevice");
    return with_dtype(a->dtype, [&](auto tag) {
      using T = decltype(tag);
      const bool wide =
          rows_aligned({&a->x, &a->input_gate, &a->recurrence_gate, &a->dout}, sizeof(T), 16);
      const RecArrays<T> p = arrays_of<T>(a);
      return wide ? run_bwd<T, kWhole>(dev, p, a->ddecay, st, what)
                  : run_bwd<T, kSingle>(dev, p, a->ddecay, st, what);
    });
  });
}

ferrum_status ferrum_gated_recurrence_step(ferrum_device* dev, const ferrum_recurrence_args* a,
                                           void* stream) {
  const char* what = "gated_recurrence_step";
  return guarded(what, [&]() -> ferrum_status {
    if (ferrum_status s = check_recurrence(dev, a, what, false)) return s;
    const int64_t n = (int64_t)a->batch * (int64_t)a->channels;
    if (a->length != 1) return invalid(what, "length must be 1, got " + std::to_string(a->length));
    if (n > 0 && (a->initial_state == nullptr || a->final_state == nullptr))
      return invalid(what, "initial_state and final_state are required");
    if (a->lengths != nullptr) return invalid(what, "lengths does not apply to one step");
    if (n == 0) return FERRUM_OK;
    DeviceGuard guard(dev->ordinal);
    if (guard.status() != cudaSuccess) return cuda_error(guard.status(), "cudaSetDevice");
    return with_dtype(a->dtype, [&](auto tag) -> ferrum_status {
      using T = decltype(tag);
      const RecArrays<T> p = arrays_of<T>(a);
      cudaStream_t st = (cudaStream_t)stream;
      const bool wide = a->channels % 4 == 0 && aligned(a->decay, 16) && aligned(a->initial_state, 16) &&
                        aligned(a->final_state, 16) &&
                        rows_aligned({&a->x, &a->input_gate, &a->recurrence_gate, &a->out}, sizeof(T),
                                     4 * sizeof(T));
      const int64_t blocks = ceil_div(wide ? n / 4 : n, kStepThreads);
      if (blocks > 0x7fffffff || a->channels > 0xffffffffull) return invalid(what, "too many values for one launch");
      launch_detail::clear_stale_error();
      if (wide)
        recurrence_step_kernel<T, 4><<<(unsigned)blocks, kStepThreads, 0, st>>>(p);
      else
        recurrence_step_kernel<T, 1><<<(unsigned)blocks, kStepThreads, 0, st>>>(p);
      return launched(what);
    });
  });
}

}  // extern "C"
