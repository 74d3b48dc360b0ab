// The loss against a vocabulary on the tensor cores, for 16-bit types.
//
// Four products share one kernel; they differ in where their operands lie and in
// what becomes of a finished tile (T tokens, D width, V vocabulary):
//   stats   x W^T  (T x V over D):  each row's largest logit and sum of exponentials
//                                   over the tile's columns, and its target's logit
//   grads   x W^T again:            G = (dloss + dlse) softmax - dloss onehot, to 16 bits
//   dx      G W    (T x D over V):  float32 sums, added over the pieces of V
//   dW      G^T x  (V x D over T):  rounded and stored
// The logits never leave the chip; G is kept for a piece of the vocabulary at a
// time, scaled so that the largest |dloss| is 2^13: float16 then holds softmax values
// down to 2^-27 in full precision, dloss may be tiny, and a target's value, nearly
// -dloss, is nearly -2^13 where all tokens weigh the same, so that its rounding to 16
// bits is none. The others' roundings have random signs: 8192 x 2048 x 32768 bf16, dx
// and dW are 0.00166 from 64 bits, of which rounding themselves is 0.00166; 16384 x 64 x
// 256, where the softmax is larger, 0.00195 and 0.00175 of 0.00165.
//
// A pair of CTAs computes a tile of 256 x 256: each stages 128 rows of A and of B
// (32 KiB a step of 64) by TMA, one thread of the leader issues 256 x 256 x 16
// products whose accumulators lie in both CTAs' TMEM, 128 rows each. There are two
// sets of accumulators (all 512 columns), so that eight warps finish one tile while
// the next is computed. 74 pairs walk the tiles; dx and dW of a piece share a launch,
// so that the last wave of one is filled by the other.
//
// 8192 x 2048 x 32768 bf16: 725 us forward (1.52 PFLOP/s; cuBLAS takes 702 for the
// logits alone), 2400 to 2550 for the gradient (1.37 to 1.29 PFLOP/s over its three
// products, at the power limit; a library product sustains 1.39). The tensor pipe is
// busy for 87 to 94 % of the cycles. What it took: one thread issues the products, so descriptors move
// by sums and tiles are numbered by 32 bits (gradient 2755 -> 2350 us); accumulators
// are read at once and released before anything is stored (16384 x 512 x 32768:
// 575 -> 386 us); an arrival that orders no memory, since one that does waits for the
// warp's stores.
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <mutex>

#include "cross_entropy.cuh"
#include "tensor_core.cuh"

namespace ferrum {
namespace seq {

namespace {
PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static std::once_flag once;
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    else
      (void)cudaGetLastError();
  });
  return fn;
}
}  // namespace

cudaError_t tensor_map(CUtensorMap* map, bool bf16, const void* base, int64_t cols, int64_t rows,
                       int64_t ld, int box_rows) {
  PFN_cuTensorMapEncodeTiled_v12000 fn = encode_fn();
  if (fn == nullptr || !mappable(base, ld, cols)) return cudaErrorNotSupported;
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  cuuint32_t box[2] = {64, (cuuint32_t)box_rows}, es[2] = {1, 1};
  const CUresult r =
      fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
         const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

namespace {

constexpr int kTile = 256, kHalf = 128, kDepth = 64, kStages = 6;
constexpr int kOperandBytes = kHalf * kDepth * 2;             // of one CTA and step
constexpr int kStageBytes = 2 * kOperandBytes;
constexpr int kEpilogueWarp = 4, kEpilogueWarps = 8;
constexpr int kThreads = 32 * (kEpilogueWarp + kEpilogueWarps);
constexpr int kSlotBytes = 32 * 128;                          // a warp's rows on their way out
// and 1024 bytes of room to align
constexpr int kSmemBytes = kStages * kStageBytes + kEpilogueWarps * kSlotBytes + 1024;
// Tokens that one chain of dW's sums takes at most. The tensor cores cut off each of its n / 16
// additions, by half a unit of 2^-23 on average, of a sum that grows as sqrt(n): n / 24 units of
// 2^-24 at its end, which is 0.17 of float16's rounding at 32768.
constexpr int64_t kChain = 32768;
// Steps of depth after which the logits of the loss are taken from TMEM and added up in
// registers, which round: a chain of width / 16 additions that are cut off shrinks its sum by
// 1.5e-8 of it each on average (1000 x 4096 x 256 bf16 in one chain: lse 1.3e-6 from 64 bits,
// loss 1.6e-6; in four 3.0e-7 and 3.6e-7; 4096 x 2048 x 32768 355 and 362 us). The gradient
// rounds to 16 bits what it makes of its logits.
constexpr int kPartSteps = 16;
constexpr uint32_t kGroup = 16;                                   // tiles of M that share a tile of N

enum Kind { kStats, kGrads, kWeights };

// One product A B^T of the extents m x n over `steps` steps of depth.
struct Product {
  int64_t m, n;
  int tiles_m, tiles_n, splits, steps, steps_per_split;
  bool a_mn;                 // A's rows run along the depth (as all of B's in kWeights)
  bool live_rows, live_depth;  // m or the depth is the number of tokens with a loss (the
                               // depth shared out to the splits)
  bool dx;                   // rows go to the tokens' places
  bool sums;                 // the result: float32 sums, a slab per split (else 16 bits)
  bool load, store_map;      // sums of earlier pieces come on top; `out` has a tensor map
  void* out;
  float* partial;            // float32 sums, rows of partial_ld
  int64_t ld, partial_ld;
};

struct Work {
  Product p[2];              // one after the other
  int count;
  int* err_flag;
  // stats
  const int64_t* targets;
  RowStat* stats;            // (half tile of N, m)
  float* at_target;
  int parts;                 // of the depth
  // gradients
  LiveTokens live;
  int known;                 // how many tokens have a loss (with those behind), if the host knows
  int64_t first;             // the piece's first word
};

struct Maps {
  CUtensorMap a, b, out;
};

// Tiles are numbered by 32 bits (the host checks): a division by 64 bits takes the
// issuing thread longer than a step of the product.
struct Place {
  int product, tm, tn, split;
};
// Extents that depend on the number `live` of tokens with a loss.
__device__ __forceinline__ int64_t rows_of(const Product& p, int live) { return p.live_rows ? live : p.m; }
__device__ __forceinline__ uint32_t tiles_m_of(const Product& p, int live) {
  return p.live_rows ? (uint32_t)(live + kTile - 1) / kTile : p.tiles_m;
}
__device__ __forceinline__ int steps_each(const Product& p, int live) {   // (as live_each())
  if (!p.live_depth) return p.steps_per_split;
  return p.splits > 1 ? (live / kDepth + p.splits - 1) / p.splits : live / kDepth;
}
// Splits that have a step of depth.
__device__ __forceinline__ int splits_of(const Product& p, int live) {
  if (!p.live_depth || p.splits == 1) return p.splits;
  const int each = steps_each(p, live);
  return (live / kDepth + each - 1) / each;
}
__device__ __forceinline__ uint32_t tiles_of(const Product& p, int live) {
  return tiles_m_of(p, live) * (uint32_t)p.tiles_n * (uint32_t)splits_of(p, live);
}
// A tile's steps of depth, from k0 up to k1.
struct Depth {
  int k0, k1;
};
__device__ __forceinline__ Depth depth_of(const Product& p, int split, int live) {
  const int each = steps_each(p, live), all = p.live_depth ? live / kDepth : p.steps;
  const int k0 = split * each, k1 = k0 + each;
  return {k0, k1 < all ? k1 : all};
}
template <int KIND>
__device__ __forceinline__ Place place_of(const Work& w, uint32_t t, int live) {
  Place q;
  q.product = 0;
  if (KIND == kWeights) {
    const uint32_t first = tiles_of(w.p[0], live);
    if (t >= first) q.product = 1, t -= first;
  }
  const Product& p = w.p[q.product];
  const uint32_t tiles_m = tiles_m_of(p, live);
  q.split = 0;
  if (KIND == kWeights && p.splits > 1) {
    const uint32_t per = tiles_m * (uint32_t)p.tiles_n;
    q.split = (int)(t / per), t %= per;
  }
  const uint32_t group = t / ((uint32_t)kGroup * p.tiles_n), first = group * kGroup;
  const uint32_t wide = tiles_m - first < kGroup ? tiles_m - first : kGroup;
  t -= first * p.tiles_n;
  q.tm = (int)(first + t % wide), q.tn = (int)(t / wide);
  return q;
}

struct Shared {
  uint64_t full[kStages], empty[kStages], done[2], drained[2];
  uint32_t tmem;
  int dead;
};

// A bounded wait; once one has run out, all others of the CTA end too.
template <class S>
__device__ __forceinline__ bool wait(S* sh, uint64_t* bar, uint32_t phase, int* err_flag) {
  if (mbar_try_wait(bar, phase)) return true;
  const uint64_t t0 = global_ns();
  while (!mbar_try_wait(bar, phase)) {
    if (*(volatile int*)&sh->dead) return false;
    if (global_ns() - t0 > kWaitTimeoutNs) {
      *(volatile int*)&sh->dead = 1;
      *(volatile int*)err_flag = kErrWaitTimeout;
      return false;
    }
  }
  return true;
}

// ---------------------------------------------------------------- epilogues
// One warp: row m (its lane's), 128 columns from n0 on, at TMEM address `acc`.
// `release` says that the accumulators have been read; it comes before the tile's
// results are stored, whose completion it would otherwise wait for.

// What an epilogue reads of its row, a tile ahead of using it.
template <int KIND>
__device__ __forceinline__ RowCoef row_ahead(const Work& w, const Place& q, int64_t m, int live) {
  RowCoef r = {0.f, 0.f, 0.f, -1};
  if constexpr (KIND == kStats) {
    if (m < w.p[0].m) {
      const int64_t at = w.targets[m];
      r.target = has_loss(at, w.p[0].n) ? (int)at : -1;
    }
  } else if constexpr (KIND == kGrads) {
    if (m < live) r = w.live.rows[m];
  } else {
    if (w.p[q.product].dx && m < live) r.target = w.live.index[m];   // (where the row goes)
  }
  return r;
}

// `more(acc)`: another part of the depth, its accumulators at `acc`, if there is one.
template <class F, class G>
__device__ void finish_stats(const Work& w, uint32_t acc, const RowCoef& row, int64_t m, int64_t n0,
                             F release, G more) {
  const Product& p = w.p[0];
  const int at = row.target - (int)n0;
  const int cols = p.n - n0 < kHalf ? (int)(p.n - n0) : kHalf;      // (may be below 0)
  if (cols <= 0) {
    do release();
    while (more(acc));
    return;
  }
  float v[4][32], hit = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) tmem_load32(acc + j * 32, v[j]);
  tmem_load_wait();
  release();
#pragma unroll 1
  while (more(acc)) {
#pragma unroll
    for (int j = 0; j < kHalf / 16; ++j) {
      float u[16];
      tmem_load16(acc + j * 16, u);
      tmem_load_wait();
#pragma unroll
      for (int i = 0; i < 16; ++i) v[j / 2][j % 2 * 16 + i] += u[i];
    }
    release();
  }
  if (cols < kHalf) {
#pragma unroll
    for (int i = 0; i < kHalf; ++i)
      if (i >= cols) v[i / 32][i % 32] = -INFINITY;
  }
  if (at >= 0 && at < kHalf) {
#pragma unroll
    for (int i = 0; i < kHalf; ++i) hit += at == i ? v[i / 32][i % 32] : 0.f;
  }
  float t4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, s4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kHalf; ++i) t4[i % 4] = fmaxf(t4[i % 4], v[i / 32][i % 32]);
  RowStat s;
  s.top = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3]));
  const float k = shift_of(s.top) * kLog2e;
#pragma unroll
  for (int i = 0; i < kHalf; ++i) s4[i % 4] += ex2(fmaf(v[i / 32][i % 32], kLog2e, -k));
  if (fabsf(s.top) > kFar && fabsf(s.top) < INFINITY) {
    s4[0] = s4[1] = s4[2] = s4[3] = 0.f;
#pragma unroll
    for (int i = 0; i < kHalf; ++i) s4[i % 4] += ex2((v[i / 32][i % 32] - s.top) * kLog2e);
  }
  s.sum = (s4[0] + s4[1]) + (s4[2] + s4[3]);
  if (m >= p.m) return;
  w.stats[n0 / kHalf * p.m + m] = s;
  if (row.target >= 0 && at >= 0 && at < kHalf) w.at_target[m] = hit;
}

// A warp's 32 rows of 64 values, on their way out through its slot of shared memory:
// rows of 128 bytes, swizzled as the tensor map has them, or single values where the
// array has no map or rows go to places of their own (`place`, the lane's row's; -1 for
// none). `rows`: those of the product.
template <class T>
__device__ __forceinline__ void put_rows(const Product& p, const CUtensorMap* map, uint8_t* slot,
                                         const float (&v)[2][32], int64_t rows, int64_t m0, int64_t n0,
                                         int place, int lane) {
  // the store that read the slot before is done with it
  if (lane == 0) bulk_wait_read_all();
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    uint4 q;
    const float* u = &v[j / 4][j % 4 * 8];
    q.x = pack_pair<T>(u[0], u[1]), q.y = pack_pair<T>(u[2], u[3]);
    q.z = pack_pair<T>(u[4], u[5]), q.w = pack_pair<T>(u[6], u[7]);
    *(uint4*)(slot + lane * 128 + ((j ^ (lane & 7)) * 16)) = q;
  }
  if (p.store_map) {
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0 && m0 < rows && n0 < p.n) {
      tma_store_tile2d(map, (int32_t)n0, (int32_t)m0, slot);
      bulk_commit();
    }
  } else {
    __syncwarp();
    const int cols = p.n - n0 < 64 ? (int)(p.n - n0) : 64;
    if (!p.dx) place = m0 + lane < rows ? (int)(m0 + lane) : -1;
    T* out = (T*)p.out + n0 + lane;
#pragma unroll 8
    for (int r = 0; r < 32; ++r) {
      const int to = __shfl_sync(0xffffffffu, place, r);
      const uint8_t* row = slot + r * 128 + lane % 8 * 2;
      const T lo = *(const T*)(row + ((lane / 8) ^ (r & 7)) * 16);
      const T hi = *(const T*)(row + ((lane / 8 + 4) ^ (r & 7)) * 16);
      if (to >= 0 && lane < cols) out[to * p.ld] = lo;
      if (to >= 0 && lane + 32 < cols) out[to * p.ld + 32] = hi;
    }
    __syncwarp();
  }
}

template <class T, class F>
__device__ void finish_grads(const Work& w, const CUtensorMap* map, uint8_t* slot, uint32_t acc,
                             const RowCoef& q, int64_t rows, int64_t m0, int64_t n0, int lane,
                             F release) {
  const Product& p = w.p[0];
  // (a target in front of the piece is below 0, whatever is taken from it)
  const int64_t at64 = (int64_t)q.target - w.first - n0;
  const int at = q.target >= 0 && at64 >= 0 && at64 < kHalf ? (int)at64 : -1;
  const float scale = softmax_scale(q.lse), lse = q.lse * scale;
  if (n0 >= p.n) release();
#pragma unroll 1
  for (int c = 0; c < kHalf; c += 64) {
    if (n0 + c >= p.n) break;
    float v[2][32];
    tmem_load32(acc + c, v[0]);
    tmem_load32(acc + c + 32, v[1]);
    tmem_load_wait();
    if (c + 64 >= kHalf || n0 + c + 64 >= p.n) release();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        v[h][i] = q.target < 0 ? 0.f : ex2(fmaf(v[h][i], scale, -lse)) * q.all;
      if (at >= c + h * 32 && at < c + h * 32 + 32) {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[h][i] -= at - c - h * 32 == i ? q.one : 0.f;
      }
    }
    put_rows<T>(p, map, slot, v, rows, m0, n0 + c, -1, lane);
  }
}

// Sums into `partial`, or with them, scaled back, to 16 bits.
template <class T, class F>
__device__ void finish_weights(const Work& w, const Product& p, const CUtensorMap* map, uint8_t* slot,
                               uint32_t acc, const RowCoef& row, int64_t rows, int64_t m0, int64_t n0,
                               int split, int lane, F release) {
  const float inv = w.live.scale[1];
  const int64_t m = m0 + lane;
  float* part = p.partial ? p.partial + ((int64_t)split * p.m + m) * p.partial_ld + n0 : nullptr;
  if (n0 >= p.n) release();
#pragma unroll 1
  for (int c = 0; c < kHalf; c += 64) {
    if (n0 + c >= p.n) break;
    float v[2][32];
    tmem_load32(acc + c, v[0]);
    tmem_load32(acc + c + 32, v[1]);
    tmem_load_wait();
    if (c + 64 >= kHalf || n0 + c + 64 >= p.n) release();
    if (p.load && m < rows) {
#pragma unroll
      for (int i = 0; i < 64; i += 4) {
        if (n0 + c + i >= p.partial_ld) continue;    // (a multiple of 8)
        const float4 b = *(const float4*)(part + c + i);
        float* u = &v[i / 32][i % 32];
        u[0] += b.x, u[1] += b.y, u[2] += b.z, u[3] += b.w;
      }
    }
    if (p.sums) {
      if (m >= rows) continue;
#pragma unroll
      for (int i = 0; i < 64; i += 4) {
        if (n0 + c + i >= p.partial_ld) continue;
        const float* u = &v[i / 32][i % 32];
        *(float4*)(part + c + i) = make_float4(u[0], u[1], u[2], u[3]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 64; ++i) v[i / 32][i % 32] *= inv;
      put_rows<T>(p, map, slot, v, rows, m0, n0 + c, row.target, lane);
    }
  }
}

// ---------------------------------------------------------------- the kernel
template <class T, int KIND>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
loss_product_kernel(const __grid_constant__ Maps maps0, const __grid_constant__ Maps maps1,
                    const __grid_constant__ Work w) {
  extern __shared__ uint8_t raw[];
  uint8_t* stages = (uint8_t*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
  __shared__ Shared sh;
  constexpr uint32_t kBlock = 64 * kDepth * 2;     // bytes between 64-value blocks of MN-major rows
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = cluster_rank();
  const uint32_t pair = blockIdx.x / 2, pairs = gridDim.x / 2;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&sh.full[i], 1), mbar_init(&sh.empty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&sh.done[i], 1), mbar_init(&sh.drained[i], 2 * kEpilogueWarps);
    sh.dead = 0;
    fence_barrier_init();
  }
  if (warp == 2) tmem_alloc_pair(&sh.tmem);
  if (warp == 3 && lane == 0) {
    map_prefetch(&maps0.a), map_prefetch(&maps0.b);
    if (KIND == kWeights) map_prefetch(&maps1.a), map_prefetch(&maps1.b);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  start_next(), await_previous();
  const int live = KIND == kStats ? 0 : (w.known ? w.known : *w.live.count);
  const uint32_t tiles = tiles_of(w.p[0], live) + (KIND == kWeights ? tiles_of(w.p[1], live) : 0);

  if (warp == 0 && lane == 0) {                    // copies
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    const uint32_t bars = map_to_rank(&sh.full[0], 0);
    auto tile = [&](auto a_mn, const Place& q) {
      constexpr bool A_MN = decltype(a_mn)::value, B_MN = KIND == kWeights;
      const Product& p = w.p[q.product];
      const CUtensorMap* map_a = q.product ? &maps1.a : &maps0.a;
      const CUtensorMap* map_b = q.product ? &maps1.b : &maps0.b;
      const int m0 = q.tm * kTile + (int)rank * kHalf, n0 = q.tn * kTile + (int)rank * kHalf;
      const int k0 = depth_of(p, q.split, live).k0, k1 = depth_of(p, q.split, live).k1;
      for (int k = k0; k < k1; ++k) {
        if (!(ok = wait(&sh, &sh.empty[stage], phase ^ 1, w.err_flag))) return;
        if (rank == 0) mbar_arrive_expect_tx(&sh.full[stage], 2 * kStageBytes);
        const uint32_t bar = bars + stage * 8;
        uint8_t* a = stages + stage * kStageBytes;
        uint8_t* b = a + kOperandBytes;
        if constexpr (A_MN) {
          pair_load(a, map_a, m0, k * kDepth, bar);
          pair_load(a + kBlock, map_a, m0 + 64, k * kDepth, bar);
        } else {
          pair_load(a, map_a, k * kDepth, m0, bar);
        }
        if constexpr (B_MN) {
          pair_load(b, map_b, n0, k * kDepth, bar);
          pair_load(b + kBlock, map_b, n0 + 64, k * kDepth, bar);
        } else {
          pair_load(b, map_b, k * kDepth, n0, bar);
        }
        if (++stage == kStages) stage = 0, phase ^= 1;
      }
    };
    for (uint32_t t = pair; ok && t < tiles; t += pairs) {
      const Place q = place_of<KIND>(w, t, live);
      if (KIND == kWeights && w.p[q.product].a_mn)
        tile(std::true_type(), q);
      else
        tile(std::false_type(), q);
    }
    // every stage's last release has arrived before this CTA may end
    for (int i = 0; ok && i < kStages; ++i) {
      ok = wait(&sh, &sh.empty[stage], phase ^ 1, w.err_flag);
      if (++stage == kStages) stage = 0, phase ^= 1;
    }
  } else if (warp == 1 && lane == 0 && rank == 0) {   // products
    // One thread issues four instructions a step of 512 cycles, so what it computes
    // per step is little: descriptors move by sums.
    int stage = 0, buf = 0;
    uint32_t phase = 0, buf_phase = 0;
    bool ok = true;
    const uint64_t first_a = operand_desc(smem_u32(stages), kBlock);
    const uint64_t first_b = operand_desc(smem_u32(stages) + kOperandBytes, kBlock);
    auto tile = [&](auto a_mn, const Place& q) {
      constexpr bool A_MN = decltype(a_mn)::value, B_MN = KIND == kWeights;
      constexpr uint32_t kIdesc = instruction_desc<T>(kTile, kTile, A_MN, B_MN);
      // 16 steps of depth: 32 bytes along a K-major row, two atoms MN-major
      constexpr uint32_t kStepA = (A_MN ? 2048 : 32) / 16, kStepB = (B_MN ? 2048 : 32) / 16;
      const Product& p = w.p[q.product];
      const int end = depth_of(p, q.split, live).k1;
      for (int k0 = depth_of(p, q.split, live).k0; k0 < end;) {
        const int k1 = KIND == kStats && end - k0 > kPartSteps ? k0 + kPartSteps : end;
        if (!(ok = wait(&sh, &sh.drained[buf], buf_phase ^ 1, w.err_flag))) return;
        tc_fence_after();
        const uint32_t acc = tmem + buf * kTile;
        for (int k = k0; k < k1; ++k) {
          if (!(ok = wait(&sh, &sh.full[stage], phase, w.err_flag))) return;
          tc_fence_after();
          const uint64_t a = first_a + stage * (kStageBytes / 16), b = first_b + stage * (kStageBytes / 16);
#pragma unroll
          for (int i = 0; i < kDepth / 16; ++i)
            mma_pair(acc, a + i * kStepA, b + i * kStepB, kIdesc, k > k0 || i > 0);
          commit_pair(&sh.empty[stage]);
          if (++stage == kStages) stage = 0, phase ^= 1;
        }
        commit_pair(&sh.done[buf]);
        if (++buf == 2) buf = 0, buf_phase ^= 1;
        k0 = k1;
      }
    };
    for (uint32_t t = pair; ok && t < tiles; t += pairs) {
      const Place q = place_of<KIND>(w, t, live);
      if (KIND == kWeights && w.p[q.product].a_mn)
        tile(std::true_type(), q);
      else
        tile(std::false_type(), q);
    }
  } else if (warp >= kEpilogueWarp) {              // finished tiles
    int buf = 0;
    uint32_t buf_phase = 0;
    // a warp reads the 32 lanes of TMEM that its number's last two bits name
    const uint32_t lanes = (uint32_t)(warp % 4) * 32, half = (uint32_t)(warp - kEpilogueWarp) / 4;
    uint8_t* slot = stages + kStages * kStageBytes + (warp - kEpilogueWarp) * kSlotBytes;
    const uint32_t drained = map_to_rank(&sh.drained[0], 0);
    Place next = {};
    RowCoef row_next = {};
    auto look_ahead = [&](uint32_t t) {
      if (t >= tiles) return;
      next = place_of<KIND>(w, t, live);
      row_next = row_ahead<KIND>(w, next, (int64_t)next.tm * kTile + rank * kHalf + lanes + lane, live);
    };
    look_ahead(pair);
    bool ok = true;
    // the next accumulators' address, once they are done
    auto await_done = [&]() -> uint32_t {
      ok = lane != 0 || wait(&sh, &sh.done[buf], buf_phase, w.err_flag);
      ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
      tc_fence_after();
      return tmem + (lanes << 16) + buf * kTile + half * kHalf;
    };
    auto release = [&] {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_at(drained + buf * 8);
    };
    for (uint32_t t = pair; t < tiles; t += pairs) {
      uint32_t acc = await_done();
      if (!ok) break;
      const Place q = next;
      const RowCoef row = row_next;
      look_ahead(t + pairs);
      const int64_t m0 = (int64_t)q.tm * kTile + rank * kHalf + lanes;
      const int64_t n0 = (int64_t)q.tn * kTile + half * kHalf;
      const CUtensorMap* out = q.product ? &maps1.out : &maps0.out;
      if constexpr (KIND == kStats) {
        int part = 0;
        auto more = [&](uint32_t& at) {
          if (++part >= w.parts) return false;
          if (++buf == 2) buf = 0, buf_phase ^= 1;
          at = await_done();
          return ok;
        };
        finish_stats(w, acc, row, m0 + lane, n0, release, more);
        if (!ok) break;
      }
      if constexpr (KIND == kGrads) finish_grads<T>(w, out, slot, acc, row, live, m0, n0, lane, release);
      if constexpr (KIND == kWeights)
        finish_weights<T>(w, w.p[q.product], out, slot, acc, row, rows_of(w.p[q.product], live), m0, n0,
                          q.split, lane, release);
      if (++buf == 2) buf = 0, buf_phase ^= 1;
    }
    if (lane == 0) bulk_wait_all();
  }
  __syncthreads();
  if (sh.dead) {     // let copies and products in flight land before their memory goes
    const uint64_t t0 = global_ns();
    while (global_ns() - t0 < 20000000ull) {
    }
  }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  if (warp == 2) tmem_free_pair(tmem);
}

// ---------------------------------------------------------------- few tokens
// With few tokens the products' time is W's way from HBM, and tiles of 256 tokens are
// mostly empty. So the sides change: 128 words are the rows of a product, the tokens
// its NT columns (32 or 64), one CTA a tile, and what shared memory is left holds
// copies of W under way (8 or 10 steps of 16 KiB). CTAs take words by units of 32, so that
// all have work of nearly one size. A warp's 32 lanes are words; values of a token
// are joined across them by exchanges that halve the columns each time, which leaves
// lane l with column l: 31 shuffles for 32 columns.
constexpr int kFewRows = 128, kUnit = 32;
constexpr int kFewThreads = 256, kFewEpilogueWarps = 4;

template <int NT>
struct FewShape {
  static constexpr int kBytesA = kFewRows * kDepth * 2, kBytesB = NT * kDepth * 2;
  static constexpr int kStage = kBytesA + kBytesB;
  static constexpr int kCount = 208 * 1024 / kStage < 12 ? 208 * 1024 / kStage : 12;
  static constexpr int kSmem = kCount * kStage + 1024;
  static constexpr int kChunks = NT / 32;
};

struct FewWork {
  int64_t tokens, vocab;
  int steps, part_steps;             // of depth, and of one of its parts
  int units, units_each;             // of words, and at most of one CTA
  int* err_flag;
  const int64_t* targets;            // stats
  RowStat* stats;                    // (CTA, token)
  float* at_target;
  const RowCoef* rows;               // grads
  void* out;                         // G transposed: (vocab, ld), tokens behind the last as zeros
  int64_t ld;
};

template <int NT>
struct FewShared {
  uint64_t full[FewShape<NT>::kCount], empty[FewShape<NT>::kCount], done[2], drained[2];
  uint32_t tmem;
  int dead;
  RowCoef rows[NT];          // (lse times `scale`)
  float scale[NT];
  RowStat stats[kFewEpilogueWarps][NT];
};

template <class F>
__device__ __forceinline__ float spread(float (&v)[32], int lane, F op) {
#pragma unroll
  for (int o = 16; o > 0; o /= 2) {
    const bool up = (lane & o) != 0;
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float keep = up ? v[i + o] : v[i], send = up ? v[i] : v[i + o];
      v[i] = op(keep, __shfl_xor_sync(0xffffffffu, send, o));
    }
  }
  return v[0];
}

template <class T, int NT, bool GRADS>
__global__ void __launch_bounds__(kFewThreads, 1)
loss_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                const __grid_constant__ FewWork w) {
  using S = FewShape<NT>;
  extern __shared__ uint8_t raw[];
  uint8_t* stages = (uint8_t*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
  __shared__ FewShared<NT> sh;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int unit0 = (int)blockIdx.x * w.units_each;
  const int unit1 = unit0 + w.units_each < w.units ? unit0 + w.units_each : w.units;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kCount; ++i) mbar_init(&sh.full[i], 1), mbar_init(&sh.empty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&sh.done[i], 1), mbar_init(&sh.drained[i], kFewEpilogueWarps);
    sh.dead = 0;
    fence_barrier_init();
  }
  if (warp == 2) tmem_alloc<2 * NT>(&sh.tmem);
  if (warp == 3 && lane == 0) map_prefetch(&map_w), map_prefetch(&map_x);
  start_next(), await_previous();
  if (threadIdx.x < NT) {
    RowCoef q = {0.f, 0.f, 0.f, -1};
    if (threadIdx.x < w.tokens) {
      if constexpr (GRADS) {
        q = w.rows[threadIdx.x];
      } else {
        const int64_t at = w.targets[threadIdx.x];
        if (has_loss(at, w.vocab)) q.target = (int)at;
      }
    }
    const float scale = softmax_scale(q.lse);
    q.lse *= scale;
    sh.rows[threadIdx.x] = q, sh.scale[threadIdx.x] = scale;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;

  if (warp == 0 && lane == 0) {                       // copies
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int u = unit0; ok && u < unit1; u += kFewRows / kUnit) {
      const int boxes = unit1 - u < kFewRows / kUnit ? unit1 - u : kFewRows / kUnit;
      for (int k = 0; k < w.steps; ++k) {
        if (!(ok = wait(&sh, &sh.empty[stage], phase ^ 1, w.err_flag))) break;
        uint8_t* a = stages + stage * S::kStage;
        mbar_arrive_expect_tx(&sh.full[stage], (uint32_t)(boxes * (S::kBytesA / 4) + S::kBytesB));
        for (int i = 0; i < boxes; ++i)
          tma_load_tile2d(a + i * (S::kBytesA / 4), &map_w, k * kDepth, (u + i) * kUnit, &sh.full[stage]);
        tma_load_tile2d(a + S::kBytesA, &map_x, k * kDepth, 0, &sh.full[stage]);
        if (++stage == S::kCount) stage = 0, phase ^= 1;
      }
    }
    for (int i = 0; ok && i < S::kCount; ++i) {
      ok = wait(&sh, &sh.empty[stage], phase ^ 1, w.err_flag);
      if (++stage == S::kCount) stage = 0, phase ^= 1;
    }
  } else if (warp == 1 && lane == 0) {                // products
    constexpr uint32_t kIdesc = instruction_desc<T>(kFewRows, NT, false, false);
    int stage = 0, buf = 0;
    uint32_t phase = 0, buf_phase = 0;
    bool ok = true;
    const uint64_t first = operand_desc(smem_u32(stages), 16);
    for (int u = unit0; ok && u < unit1; u += kFewRows / kUnit) {
      for (int k0 = 0; ok && k0 < w.steps; k0 += w.part_steps) {
        const int k1 = w.steps - k0 > w.part_steps ? k0 + w.part_steps : w.steps;
        if (!(ok = wait(&sh, &sh.drained[buf], buf_phase ^ 1, w.err_flag))) break;
        tc_fence_after();
        for (int k = k0; k < k1; ++k) {
          if (!(ok = wait(&sh, &sh.full[stage], phase, w.err_flag))) break;
          tc_fence_after();
          const uint64_t a = first + stage * (S::kStage / 16), b = a + S::kBytesA / 16;
#pragma unroll
          for (int i = 0; i < kDepth / 16; ++i)
            mma_one(tmem + buf * NT, a + i * 2, b + i * 2, kIdesc, k > k0 || i > 0);
          commit_one(&sh.empty[stage]);
          if (++stage == S::kCount) stage = 0, phase ^= 1;
        }
        if (!ok) break;
        commit_one(&sh.done[buf]);
        if (++buf == 2) buf = 0, buf_phase ^= 1;
      }
    }
  } else if (warp >= 4) {                             // finished tiles
    int buf = 0;
    uint32_t buf_phase = 0;
    const int part = warp - 4;
    RowStat run[S::kChunks];
#pragma unroll
    for (int c = 0; c < S::kChunks; ++c) run[c] = {-INFINITY, 0.f};
    for (int u = unit0; u < unit1; u += kFewRows / kUnit) {
      float sums[S::kChunks][32];
      bool ok = true;
      for (int k0 = 0; k0 < w.steps; k0 += w.part_steps) {
        ok = lane != 0 || wait(&sh, &sh.done[buf], buf_phase, w.err_flag);
        ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
        if (!ok) break;
        tc_fence_after();
        const uint32_t acc = tmem + ((uint32_t)part * 32 << 16) + buf * NT;
#pragma unroll
        for (int c = 0; c < S::kChunks; ++c) {
          float v[32];
          tmem_load32(acc + c * 32, v);
          tmem_load_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) sums[c][i] = k0 == 0 ? v[i] : sums[c][i] + v[i];
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.drained[buf]);
        if (++buf == 2) buf = 0, buf_phase ^= 1;
      }
      if (!ok) break;
      // (a part without words of this CTA's holds what an earlier tile left)
      const int64_t word = (int64_t)(u + part) * kUnit + lane;
      const bool mine = u + part < unit1 && word < w.vocab;
#pragma unroll
      for (int c = 0; c < S::kChunks; ++c) {
        float (&v)[32] = sums[c];
        if constexpr (GRADS) {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const RowCoef q = sh.rows[c * 32 + i];
            const float g = ex2(fmaf(v[i], sh.scale[c * 32 + i], -q.lse)) * q.all - (q.target == word ? q.one : 0.f);
            v[i] = q.target < 0 ? 0.f : g;
          }
          if (mine) {
            T* out = (T*)w.out + word * w.ld + c * 32;
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              float o[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) o[j] = v[i + j];
              store_vec<T, 8>(out + i, o);
            }
            if (NT == 32) {          // (rows are of 64 values at least)
              const float zero[8] = {};
#pragma unroll
              for (int i = 32; i < 64; i += 8) store_vec<T, 8>(out + i, zero);
            }
          }
        } else {
          if (!mine) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = -INFINITY;
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (sh.rows[c * 32 + i].target == word) w.at_target[c * 32 + i] = v[i];
          }
          float m[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) m[i] = v[i];
          const float top = spread(m, lane, [](float a, float b) { return fmaxf(a, b); });
          const float shift = shift_of(top), shift2 = shift * kLog2e;
          if (__any_sync(0xffffffffu, fabsf(shift) > kFar)) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {         // (other tokens as below)
              const float from = __shfl_sync(0xffffffffu, shift, i), from2 = __shfl_sync(0xffffffffu, shift2, i);
              v[i] = ex2(fabsf(from) > kFar ? (v[i] - from) * kLog2e : fmaf(v[i], kLog2e, -from2));
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              v[i] = ex2(fmaf(v[i], kLog2e, -__shfl_sync(0xffffffffu, shift2, i)));
          }
          const float sum = spread(v, lane, [](float a, float b) { return a + b; });
          run[c] = join(run[c], {top, sum});
        }
      }
    }
    if constexpr (!GRADS) {
#pragma unroll
      for (int c = 0; c < S::kChunks; ++c) sh.stats[part][c * 32 + lane] = run[c];
    }
  }
  __syncthreads();
  if (!GRADS && threadIdx.x < NT && threadIdx.x < w.tokens) {
    RowStat s = sh.stats[0][threadIdx.x];
    for (int i = 1; i < kFewEpilogueWarps; ++i) s = join(s, sh.stats[i][threadIdx.x]);
    w.stats[(int64_t)blockIdx.x * w.tokens + threadIdx.x] = s;
  }
  if (sh.dead) {     // let copies and products in flight land before their memory goes
    const uint64_t t0 = global_ns();
    while (global_ns() - t0 < 20000000ull) {
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 2) tmem_free<2 * NT>(tmem);
}

// ---------------------------------------------------------------- host
int pair_count() { return sm_count() / 2; }

Product product_of(int64_t m, int64_t n, int64_t depth, int splits = 1) {
  Product p = {};
  p.m = m, p.n = n;
  p.tiles_m = (int)ceil_div(m, kTile), p.tiles_n = (int)ceil_div(n, kTile);
  p.steps = (int)ceil_div(depth, kDepth);
  p.steps_per_split = (int)ceil_div(p.steps, splits);
  p.splits = (int)ceil_div(p.steps, p.steps_per_split);      // no empty one
  return p;
}

template <class T, int KIND>
ferrum_status run(const Maps& m0, const Maps& m1, const Work& w, bool first, cudaStream_t stream,
                  const char* what) {
  static std::atomic<uint64_t> smem_done{0};
  auto kernel = loss_product_kernel<T, KIND>;
  cudaError_t e = launch_detail::ensure_smem(kernel, kSmemBytes, smem_done);
  if (e != cudaSuccess) return cuda_error(e, what);
  int64_t tiles = 0;
  for (int i = 0; i < w.count; ++i)
    tiles += (int64_t)w.p[i].tiles_m * w.p[i].tiles_n * w.p[i].splits;
  if (tiles > 0x7fffffff) return invalid(what, "too many tiles for one launch");
  const int grid = 2 * (int)std::min<int64_t>(tiles, pair_count());
  return start(what, first, kernel, grid, kThreads, kSmemBytes, stream, m0, m1, w);
}

template <class T>
constexpr bool is_bf16() { return std::is_same<T, __nv_bfloat16>::value; }

// Up to so many tokens the sides change. Forward and gradient, us, with tiles of 256
// tokens and with the sides changed: 8 x 4096 x 131072 267, 607 and 195, 587;
// 40 x 2048 x 32000 40.8, 114 and 39.3, 103; 64 x 256 x 2000 13.9, 27 and 15.4, 23.5;
// 64 x 512 x 8000 16.9, 49 and 14.8, 43; 64 x 2048 x 32000 40.8, 112 and 39.3, 103;
// 64 x 4096 x 32000 61.4, 180 and 63.1, 172; 64 x 4096 x 131072 198, 610 and 200, 595.
// 100 x 2048 x 32000 37.4, 113 and 43.0, 111.
constexpr int64_t kFewTokens = 64;

// Launches the kernel for few tokens; `ctas` (of the statistics) is set.
template <class T, bool GRADS>
ferrum_status run_few(const Matrix<T>& wt, const Matrix<T>& x, int64_t width, FewWork w, int& ctas,
                      bool first, cudaStream_t stream, const char* what) {
  w.steps = (int)ceil_div(width, kDepth), w.units = (int)ceil_div(w.vocab, kUnit);
  w.part_steps = GRADS ? w.steps : kPartSteps;
  w.units_each = (int)ceil_div(w.units, 2 * pair_count());
  ctas = (int)ceil_div(w.units, w.units_each);
  auto go = [&](auto n) -> ferrum_status {
    constexpr int NT = decltype(n)::value;
    static std::atomic<uint64_t> smem_done{0};
    CUtensorMap mw, mx;
    cudaError_t e = tensor_map(&mw, is_bf16<T>(), wt.p, width, w.vocab, wt.ld, kUnit);
    if (e == cudaSuccess) e = tensor_map(&mx, is_bf16<T>(), x.p, width, w.tokens, x.ld, NT);
    if (e != cudaSuccess) return cuda_error(e, "tensor map");
    auto kernel = loss_few_kernel<T, NT, GRADS>;
    e = launch_detail::ensure_smem(kernel, FewShape<NT>::kSmem, smem_done);
    if (e != cudaSuccess) return cuda_error(e, what);
    return start(what, first, kernel, ctas, kFewThreads, FewShape<NT>::kSmem, stream, mw, mx, w);
  };
  return w.tokens <= 32 ? go(std::integral_constant<int, 32>()) : go(std::integral_constant<int, 64>());
}

template <class T>
ferrum_status fwd(ferrum_device* dev, const ferrum_cross_entropy_args* a, cudaStream_t stream,
                  const char* what) {
  const int64_t n = (int64_t)a->tokens, d = (int64_t)a->width, v = (int64_t)a->vocab;
  const bool copy_x = !mappable(a->x, a->x_stride, d), copy_w = !mappable(a->weight, a->weight_stride, d);
  const bool few = n <= kFewTokens;
  const int64_t ld = padded(d);
  int parts = few ? 2 * pair_count() : (int)ceil_div(v, kHalf);      // of each row's statistics
  const size_t copies = (size_t)((copy_x ? n : 0) + (copy_w ? v : 0)) * ld * 2;
  PoolBuffer ws(dev, copies + (size_t)(parts * n) * sizeof(RowStat) + (size_t)n * 4, stream);
  if (ws.status() != cudaSuccess) return cuda_error(ws.status(), "workspace");
  uint8_t* at = ws.as<uint8_t>();
  Matrix<T> x = {(const T*)a->x, a->x_stride}, wt = {(const T*)a->weight, a->weight_stride};
  if (copy_x) {
    if (ferrum_status s = copied(x, d, n, at, true, stream, what)) return s;
  }
  if (copy_w) {
    if (ferrum_status s = copied(wt, d, v, at, !copy_x, stream, what)) return s;
  }
  const bool first = !copy_x && !copy_w;
  RowStat* stats = (RowStat*)at;
  float* at_target = (float*)(stats + parts * n);
  if (few) {
    FewWork w = {};
    w.tokens = n, w.vocab = v, w.err_flag = dev->err_flag, w.targets = a->targets;
    w.stats = stats, w.at_target = at_target;
    if (ferrum_status s = run_few<T, false>(wt, x, d, w, parts, first, stream, what)) return s;
  } else {
    Maps m = {};
    cudaError_t e = tensor_map(&m.a, is_bf16<T>(), x.p, d, n, x.ld, kHalf);
    if (e == cudaSuccess) e = tensor_map(&m.b, is_bf16<T>(), wt.p, d, v, wt.ld, kHalf);
    if (e != cudaSuccess) return cuda_error(e, "tensor map");
    Work w = {};
    w.p[0] = product_of(n, v, d), w.count = 1;
    w.err_flag = dev->err_flag, w.targets = a->targets;
    w.stats = stats, w.at_target = at_target;
    w.parts = (int)ceil_div(w.p[0].steps, kPartSteps);
    if (ferrum_status s = run<T, kStats>(m, m, w, first, stream, what)) return s;
  }
  return finish_loss(stats, parts, at_target, a, stream, what);
}

// Words of a piece of the vocabulary: 256 MiB of G, but no fewer than 4096 (gradient of
// 8192 x 2048 x 32768 with 128 and 256 MiB: 2466 and 2350 us; every piece but the first
// reads dx's sums again).
int64_t piece_of(int64_t tokens, int64_t vocab) {
  const int64_t n = std::max<int64_t>(((int64_t)1 << 27) / tokens / kTile * kTile, 4096);
  return std::min(n, ceil_div(vocab, 64) * 64);
}

template <class T>
ferrum_status bwd(ferrum_device* dev, const ferrum_cross_entropy_args* a, cudaStream_t stream,
                  const char* what) {
  const int64_t n = (int64_t)a->tokens, d = (int64_t)a->width, v = (int64_t)a->vocab;
  const bool copy_w = !mappable(a->weight, a->weight_stride, d);
  // With few tokens G lies the other way: (vocabulary, 64 tokens).
  const bool few = n <= kFewTokens;
  const int64_t ld = padded(d), piece = few ? v : piece_of(n, v), g_ld = few ? kDepth : piece;
  const bool one_piece = piece >= v;
  // Few tokens make few tiles of dx: its depth is split so that all pairs work.
  const int64_t dx_tiles = ceil_div(n, kTile) * ceil_div(d, kTile);
  const int want = (int)std::max<int64_t>(
      1, std::min<int64_t>(pair_count() / dx_tiles, ceil_div(std::min(piece, v), 4 * kDepth)));
  const int splits = product_of(n, d, std::min(piece, v), want).splits;
  const int64_t rows = ceil_div(n, kDepth) * kDepth;    // room for all tokens
  // So are the tokens of few tiles of dW, from 4096 on and 1024 at least in a split, since its
  // sums take a launch to join (us without and with splits: 1500 x 256 x 500 32.5 and 37.6,
  // 2500 x 256 x 500 37.6 and 40.2, 4096 x 1024 x 1000 68.7 and 57.5, 16384 x 64 x 256 96.6 and
  // 43.5, with splits of 256 tokens 60), and those of a long chain.
  const int64_t dw_tiles = ceil_div(std::min(piece, v), kTile) * ceil_div(d, kTile);
  const int64_t dw_want = std::max(n < 4096 ? 1 : std::min<int64_t>(pair_count() / dw_tiles, n / 1024),
                                   ceil_div(n, kChain));
  const int dw_splits = few ? 1 : product_of(1, 1, rows, (int)dw_want).splits;
  const bool need_sums = splits > 1 || !one_piece;
  auto round = [](int64_t b) { return (size_t)((b + 255) / 256 * 256); };
  const size_t x_bytes = round(n * ld * 2), w_bytes = copy_w ? round(v * ld * 2) : 0;
  const size_t g_bytes = round((few ? v : rows) * g_ld * 2);
  const size_t sum_bytes = need_sums ? round(splits * rows * ld * 4) : 0;
  const size_t dw_bytes = dw_splits > 1 ? round(dw_splits * std::min(piece, v) * ld * 4) : 0;
  const size_t row_bytes = round(rows * sizeof(RowCoef)), index_bytes = round(rows * 4);
  PoolBuffer ws(dev, x_bytes + w_bytes + g_bytes + sum_bytes + dw_bytes + row_bytes + index_bytes + 256, stream);
  if (ws.status() != cudaSuccess) return cuda_error(ws.status(), "workspace");
  uint8_t* at = ws.as<uint8_t>();
  LiveTokens live;
  live.round = kDepth, live.x_rows = n;      // (the tensor maps end there)
  live.scale = (float*)at, live.count = (int*)(at + 16);
  live.rows = (RowCoef*)(at += 256), live.index = (int*)(at += row_bytes);
  at += index_bytes;
  T* x = (T*)at;
  at += x_bytes;
  T* g = (T*)at;
  at += g_bytes;
  float* sums = need_sums ? (float*)at : nullptr;
  float* dw_sums = (float*)(at += sum_bytes);
  at += dw_bytes;
  Matrix<T> wt = {(const T*)a->weight, a->weight_stride};
  if (ferrum_status s = start(what, true, prepare_kernel<T>, blocks_to_prepare(n, ld * 2), 1024, 0, stream,
                              (const T*)a->x, a->x_stride, d, x, ld, n, v, a->targets,
                              (const float*)a->lse, a->dloss, a->dlse, live, (T*)a->dx, a->dx_stride))
    return s;
  if (copy_w) {
    if (ferrum_status s = copied(wt, d, v, at, false, stream, what)) return s;
  }

  const bool dw_map = mappable(a->dweight, a->dweight_stride, d);
  for (int64_t first = 0; first < v; first += piece) {
    const int64_t words = std::min(piece, v - first);
    const bool last = first + words == v;
    const T* wp = wt.p + first * wt.ld;
    T* dw = (T*)a->dweight + first * a->dweight_stride;
    Maps logits = {}, mx = {}, mw = {};
    cudaError_t e = cudaSuccess;
    auto map = [&](CUtensorMap& m, const void* p, int64_t cols, int64_t rows, int64_t pitch, int box) {
      if (e == cudaSuccess) e = tensor_map(&m, is_bf16<T>(), p, cols, rows, pitch, box);
    };
    if (!few) {
      map(logits.a, x, d, n, ld, kHalf), map(logits.b, wp, d, words, wt.ld, kHalf);
      map(logits.out, g, words, rows, g_ld, 32);
    }
    if (few)
      map(mx.a, g, g_ld, words, g_ld, kDepth), map(mw.a, g, g_ld, words, g_ld, kHalf);
    else
      map(mx.a, g, words, rows, g_ld, kHalf), map(mw.a, g, words, rows, g_ld, kDepth);
    map(mx.b, wp, d, words, wt.ld, kDepth), map(mw.b, x, d, n, ld, kDepth);
    if (dw_map) map(mw.out, dw, d, words, a->dweight_stride, 32);
    if (e != cudaSuccess) return cuda_error(e, "tensor map");
    Work w = {};
    w.err_flag = dev->err_flag, w.live = live, w.first = first;
    w.known = rows == kDepth ? kDepth : 0;
    if (few) {
      FewWork f = {};
      int ctas = 0;
      f.tokens = n, f.vocab = v, f.err_flag = dev->err_flag, f.rows = live.rows, f.out = g, f.ld = g_ld;
      if (ferrum_status s = run_few<T, true>(wt, Matrix<T>{x, ld}, d, f, ctas, false, stream, what)) return s;
    } else {
      w.p[0] = product_of(rows, words, d), w.count = 1;
      w.p[0].store_map = w.p[0].live_rows = true;
      w.p[0].out = g;
      if (ferrum_status s = run<T, kGrads>(logits, logits, w, false, stream, what)) return s;
    }

    Product px = product_of(rows, d, words, splits), pw = product_of(words, d, few ? g_ld : rows, dw_splits);
    px.live_rows = px.dx = true, pw.live_depth = !few;
    px.partial = sums, px.partial_ld = ld;
    px.load = first > 0, px.sums = splits > 1 || !last;
    px.out = a->dx, px.ld = a->dx_stride;
    (few ? px : pw).a_mn = true;
    pw.out = dw, pw.ld = a->dweight_stride, pw.store_map = dw_map;
    if (dw_splits > 1) pw.sums = true, pw.partial = dw_sums, pw.partial_ld = ld;
    // the product of the longer tiles first, so that the last ones are short
    const bool x_first = px.steps_per_split >= pw.steps_per_split;
    w.p[0] = x_first ? px : pw, w.p[1] = x_first ? pw : px, w.count = 2;
    if (ferrum_status s = run<T, kWeights>(x_first ? mx : mw, x_first ? mw : mx, w, false, stream, what)) return s;
    if (dw_splits > 1) {
      const int64_t grid = std::min<int64_t>(ceil_div(words * ld / 4, 256), sm_count() * 16);
      if (ferrum_status s = start(what, false, finish_dw_kernel<T>, grid, 256, 0, stream, (const float*)dw_sums,
                                  dw_splits, kDepth, ld, words, d, live, dw, a->dweight_stride))
        return s;
    }
  }
  if (splits > 1)
    return start(what, false, finish_dx_kernel<T>, std::min<int64_t>(ceil_div(n * ld / 4, 256), sm_count() * 16),
                 256, 0, stream, (const float*)sums, splits, ld, rows, d, live, (T*)a->dx, a->dx_stride);
  return FERRUM_OK;
}

}  // namespace

ferrum_status loss_fwd_tc(ferrum_device* dev, const ferrum_cross_entropy_args* a,
                          cudaStream_t stream, const char* what) {
  return a->dtype == FERRUM_F16 ? fwd<__half>(dev, a, stream, what)
                                : fwd<__nv_bfloat16>(dev, a, stream, what);
}

ferrum_status loss_bwd_tc(ferrum_device* dev, const ferrum_cross_entropy_args* a,
                          cudaStream_t stream, const char* what) {
  return a->dtype == FERRUM_F16 ? bwd<__half>(dev, a, stream, what)
                                : bwd<__nv_bfloat16>(dev, a, stream, what);
}

}  // namespace seq
}  // namespace ferrum
