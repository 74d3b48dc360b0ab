// The loss against a vocabulary on the tensor cores, for 16-bit types.
//
// Four products share one kernel, which differ in where their operands lie and
// in what becomes of a finished tile (T tokens, D width, V vocabulary):
//   stats   x W^T  (T x V over D):  each row's largest logit and sum of exponentials
//                                   over the tile's columns, and its target's logit
//   grads   x W^T again:            G = (dloss + dlse) softmax - dloss onehot, to 16 bits
//   dx      G W    (T x D over V):  float32 sums, added over the pieces of V
//   dW      G^T x  (V x D over T):  rounded and stored
// The logits never leave the chip; G is kept for a piece of the vocabulary at a
// time. Rounding G to the type of x moves a gradient by as much as rounding the
// gradient itself does, no more: its terms' errors have random signs. G is scaled
// by a power of two that puts the largest |dloss| at 2^13 to 2^14, so that float16
// holds softmax values down to 2^-27 in full precision and dloss may be tiny.
//
// A pair of CTAs computes a tile of 256 x 256: each stages 128 rows of A and of B
// (32 KiB a step of 64) by TMA, one thread of the leader issues 256 x 256 x 16
// products whose accumulators lie in both CTAs' TMEM, 128 rows each. There are two
// sets of accumulators (all 512 columns), so that four warps finish one tile while
// the next is computed. 74 pairs walk the tiles.
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
constexpr int kThreads = 256, kEpilogueWarp = 4;
constexpr int kSmemBytes = kStages * kStageBytes + 1024;      // and room to align
constexpr int kGroup = 16;                                    // tiles of M that share a tile of N

enum Kind { kStats, kGrads, kDx, kDw };

// What a row needs to turn its logits into G: scaled gradients of its logits'
// sum and of its loss, lse in units of ln 2, and its target (-1 without a loss).
struct RowCoef {
  float all, one, lse2;
  int target;
};

struct Product {
  int64_t m, n;              // extents of the result
  int tiles_m, tiles_n, splits, steps, steps_per_split;
  int* err_flag;
  // stats
  const int64_t* targets;
  RowStat* stats;            // (tile of N, m)
  float* at_target;
  // grads
  const RowCoef* rows;
  int64_t first;             // the piece's first word
  // grads: G; dx: the float32 sums (a slab per split); dW: dweight
  void* out;
  int64_t ld;
  bool add;
  const float* scale;        // {2^s, 2^-s}
};

struct Place {
  int tm, tn, split;
};
__device__ __forceinline__ Place place_of(const Product& p, int64_t t) {
  const int64_t per = (int64_t)p.tiles_m * p.tiles_n;
  Place q;
  q.split = (int)(t / per);
  t %= per;
  const int64_t group = t / ((int64_t)kGroup * p.tiles_n);
  const int first = (int)group * kGroup;
  const int wide = p.tiles_m - first < kGroup ? p.tiles_m - first : kGroup;
  t -= group * kGroup * p.tiles_n;
  q.tm = first + (int)(t % wide), q.tn = (int)(t / wide);
  return q;
}

struct Shared {
  uint64_t full[kStages], empty[kStages], done[2], drained[2];
  uint32_t tmem;
  int dead;
};

// A bounded wait; once one has run out, all others of the CTA end too.
__device__ __forceinline__ bool wait(Shared* sh, uint64_t* bar, uint32_t phase, int* err_flag) {
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
// One warp: rows m0 + lane, columns n0 .. n0 + 255 of a tile at TMEM address `acc`.

__device__ void finish_stats(const Product& p, uint32_t acc, int64_t m, int64_t n0, int tn) {
  const bool row = m < p.m;
  const int64_t target = row ? p.targets[m] : -1;
  const int at = target >= n0 && target < n0 + kTile && target < p.n ? (int)(target - n0) : -1;
  const int cols = p.n - n0 < kTile ? (int)(p.n - n0) : kTile;
  RowStat s = {-INFINITY, 0.f};
  float hit = 0.f;
#pragma unroll 1
  for (int c = 0; c < kTile; c += 32) {
    if (c >= cols) break;
    float v[32];
    tmem_load32(acc + c, v);
    tmem_load_wait();
    if (c + 32 > cols) {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (c + i >= cols) v[i] = -INFINITY;
    }
    if (at >= c && at < c + 32) {
#pragma unroll
      for (int i = 0; i < 32; ++i) hit += at - c == i ? v[i] : 0.f;
    }
    float top = v[0];
#pragma unroll
    for (int i = 1; i < 32; ++i) top = fmaxf(top, v[i]);
    top = fmaxf(top, s.top);
    const float k = shift_of(top) * kLog2e;
    float sum = s.top == -INFINITY ? s.sum : s.sum * ex2(fmaf(shift_of(s.top), kLog2e, -k));
#pragma unroll
    for (int i = 0; i < 32; ++i) sum += ex2(fmaf(v[i], kLog2e, -k));
    s.top = top, s.sum = sum;
  }
  if (!row) return;
  p.stats[(int64_t)tn * p.m + m] = s;
  if (at >= 0) p.at_target[m] = hit;
}

template <class T>
__device__ void finish_grads(const Product& p, uint32_t acc, int64_t m, int64_t n0) {
  const bool row = m < p.m;
  RowCoef q = {0.f, 0.f, 0.f, -1};
  if (row) q = p.rows[m];
  const int64_t at64 = (int64_t)q.target - p.first - n0;
  const int at = q.target >= 0 && at64 >= 0 && at64 < kTile ? (int)at64 : -1;
  T* out = (T*)p.out + m * p.ld + n0;
#pragma unroll 1
  for (int c = 0; c < kTile; c += 32) {
    if (n0 + c >= p.ld) break;          // (ld is a multiple of 32)
    float v[32];
    tmem_load32(acc + c, v);
    tmem_load_wait();
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = q.target < 0 ? 0.f : ex2(fmaf(v[i], kLog2e, -q.lse2)) * q.all;
    if (at >= c && at < c + 32) {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] -= at - c == i ? q.one : 0.f;
    }
    if (row) {
#pragma unroll
      for (int i = 0; i < 32; i += 8) {
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = v[i + j];
        store_vec<T, 8>(out + c + i, w);
      }
    }
  }
}

__device__ void finish_dx(const Product& p, uint32_t acc, int64_t m, int64_t n0, int split) {
  float* out = (float*)p.out + ((int64_t)split * p.m + m) * p.ld + n0;
#pragma unroll 1
  for (int c = 0; c < kTile; c += 32) {
    float v[32];
    tmem_load32(acc + c, v);
    tmem_load_wait();
    if (m >= p.m) continue;
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      if (n0 + c + i >= p.ld) continue;    // (ld is a multiple of 8)
      float4* o = (float4*)(out + c + i);
      float4 w = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
      if (p.add) {
        const float4 b = *o;
        w.x += b.x, w.y += b.y, w.z += b.z, w.w += b.w;
      }
      *o = w;
    }
  }
}

template <class T>
__device__ void finish_dw(const Product& p, uint32_t acc, int64_t m, int64_t n0) {
  const float inv = p.scale[1];
  T* out = (T*)p.out + m * p.ld + n0;
  const bool wide = p.ld % 8 == 0 && (uintptr_t)p.out % 16 == 0;
#pragma unroll 1
  for (int c = 0; c < kTile; c += 32) {
    if (n0 + c >= p.n) break;
    float v[32];
    tmem_load32(acc + c, v);
    tmem_load_wait();
    if (m >= p.m) continue;
#pragma unroll
    for (int i = 0; i < 32; i += 8) {
      float w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = v[i + j] * inv;
      const int64_t left = p.n - (n0 + c + i);
      if (wide && left >= 8) {
        store_vec<T, 8>(out + c + i, w);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j < left) out[c + i + j] = from_f<T>(w[j]);
      }
    }
  }
}

// ---------------------------------------------------------------- the kernel
// A is K-major (rows of the depth) in all products but dW's; B in stats and grads.
template <class T, int KIND>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
loss_product_kernel(const __grid_constant__ CUtensorMap map_a,
                    const __grid_constant__ CUtensorMap map_b, Product p) {
  constexpr bool A_MN = KIND == kDw, B_MN = KIND == kDx || KIND == kDw;
  constexpr uint32_t kIdesc = instruction_desc<T, A_MN, B_MN>(kTile, kTile);
  constexpr uint32_t kBlock = 64 * kDepth * 2;     // bytes between 64-value blocks of MN-major rows
  extern __shared__ uint8_t raw[];
  uint8_t* stages = (uint8_t*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
  __shared__ Shared sh;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = cluster_rank();
  const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n * p.splits;
  const int64_t pair = blockIdx.x / 2, pairs = gridDim.x / 2;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&sh.full[i], 1), mbar_init(&sh.empty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&sh.done[i], 1), mbar_init(&sh.drained[i], 8);
    sh.dead = 0;
    fence_barrier_init();
  }
  if (warp == 2) tmem_alloc_pair(&sh.tmem);
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;

  if (warp == 0 && lane == 0) {                    // copies
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int64_t t = pair; ok && t < tiles; t += pairs) {
      const Place q = place_of(p, t);
      const int m0 = q.tm * kTile + (int)rank * kHalf, n0 = q.tn * kTile + (int)rank * kHalf;
      const int k0 = q.split * p.steps_per_split;
      const int k1 = k0 + p.steps_per_split < p.steps ? k0 + p.steps_per_split : p.steps;
      for (int k = k0; k < k1; ++k) {
        if (!(ok = wait(&sh, &sh.empty[stage], phase ^ 1, p.err_flag))) break;
        if (rank == 0) mbar_arrive_expect_tx(&sh.full[stage], 2 * kStageBytes);
        const uint32_t bar = map_to_rank(&sh.full[stage], 0);
        uint8_t* a = stages + stage * kStageBytes;
        uint8_t* b = a + kOperandBytes;
        if constexpr (A_MN) {
          pair_load(a, &map_a, m0, k * kDepth, bar);
          pair_load(a + kBlock, &map_a, m0 + 64, k * kDepth, bar);
        } else {
          pair_load(a, &map_a, k * kDepth, m0, bar);
        }
        if constexpr (B_MN) {
          pair_load(b, &map_b, n0, k * kDepth, bar);
          pair_load(b + kBlock, &map_b, n0 + 64, k * kDepth, bar);
        } else {
          pair_load(b, &map_b, k * kDepth, n0, bar);
        }
        if (++stage == kStages) stage = 0, phase ^= 1;
      }
    }
    // every stage's last release has arrived before this CTA may end
    for (int i = 0; ok && i < kStages; ++i) {
      ok = wait(&sh, &sh.empty[stage], phase ^ 1, p.err_flag);
      if (++stage == kStages) stage = 0, phase ^= 1;
    }
  } else if (warp == 1 && lane == 0 && rank == 0) {   // products
    int stage = 0, buf = 0;
    uint32_t phase = 0, buf_phase = 0;
    bool ok = true;
    for (int64_t t = pair; ok && t < tiles; t += pairs) {
      const Place q = place_of(p, t);
      const int k0 = q.split * p.steps_per_split;
      const int k1 = k0 + p.steps_per_split < p.steps ? k0 + p.steps_per_split : p.steps;
      if (!(ok = wait(&sh, &sh.drained[buf], buf_phase ^ 1, p.err_flag))) break;
      tc_fence_after();
      for (int k = k0; k < k1; ++k) {
        if (!(ok = wait(&sh, &sh.full[stage], phase, p.err_flag))) break;
        tc_fence_after();
        const uint32_t a = smem_u32(stages + stage * kStageBytes), b = a + kOperandBytes;
#pragma unroll
        for (int i = 0; i < kDepth / 16; ++i) {
          // 16 steps of depth: 32 bytes along a K-major row, two atoms MN-major
          const uint64_t da = operand_desc(a + i * (A_MN ? 2048 : 32), A_MN ? kBlock : 16);
          const uint64_t db = operand_desc(b + i * (B_MN ? 2048 : 32), B_MN ? kBlock : 16);
          mma_pair(tmem + buf * kTile, da, db, kIdesc, k > k0 || i > 0);
        }
        commit_pair(&sh.empty[stage]);
        if (++stage == kStages) stage = 0, phase ^= 1;
      }
      if (!ok) break;
      commit_pair(&sh.done[buf]);
      if (++buf == 2) buf = 0, buf_phase ^= 1;
    }
  } else if (warp >= kEpilogueWarp) {              // finished tiles
    int buf = 0;
    uint32_t buf_phase = 0;
    const uint32_t lanes = (uint32_t)(warp - kEpilogueWarp) * 32;
    for (int64_t t = pair; t < tiles; t += pairs) {
      const Place q = place_of(p, t);
      bool ok = lane != 0 || wait(&sh, &sh.done[buf], buf_phase, p.err_flag);
      ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
      if (!ok) break;
      tc_fence_after();
      const uint32_t acc = tmem + (lanes << 16) + buf * kTile;
      const int64_t m = (int64_t)q.tm * kTile + rank * kHalf + lanes + lane;
      const int64_t n0 = (int64_t)q.tn * kTile;
      if constexpr (KIND == kStats) finish_stats(p, acc, m, n0, q.tn);
      if constexpr (KIND == kGrads) finish_grads<T>(p, acc, m, n0);
      if constexpr (KIND == kDx) finish_dx(p, acc, m, n0, q.split);
      if constexpr (KIND == kDw) finish_dw<T>(p, acc, m, n0);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_at(map_to_rank(&sh.drained[buf], 0));
      if (++buf == 2) buf = 0, buf_phase ^= 1;
    }
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

// ---------------------------------------------------------------- small kernels

// A row's loss from its tiles' statistics: 32 rows by 8 strands of tiles a block,
// joined in a fixed order.
__global__ void __launch_bounds__(256)
finish_loss_kernel(const RowStat* __restrict__ stats, int tiles, int64_t tokens, int64_t vocab,
                   const int64_t* __restrict__ targets, const float* __restrict__ at_target,
                   float* __restrict__ loss, float* __restrict__ lse) {
  __shared__ RowStat part[8][32];
  const int x = threadIdx.x % 32, y = threadIdx.x / 32;
  const int64_t t = (int64_t)blockIdx.x * 32 + x;
  RowStat s = {-INFINITY, 0.f};
  if (t < tokens) {
#pragma unroll 4
    for (int i = y; i < tiles; i += 8) s = join(s, stats[(int64_t)i * tokens + t]);
  }
  part[y][x] = s;
  __syncthreads();
  if (y != 0 || t >= tokens) return;
  for (int i = 1; i < 8; ++i) s = join(s, part[i][x]);
  const bool counts = has_loss(targets[t], vocab);
  const float v = lse_of(s);
  lse[t] = counts ? v : 0.f;
  loss[t] = counts ? v - at_target[t] : 0.f;
}

// Scale of G and every row's coefficients, in one block.
__global__ void __launch_bounds__(1024)
row_coefs_kernel(int64_t tokens, int64_t vocab, const int64_t* __restrict__ targets,
                 const float* __restrict__ lse, const float* __restrict__ dloss,
                 const float* __restrict__ dlse, RowCoef* __restrict__ rows, float* scale) {
  __shared__ float part[32];
  float top = 0.f;
  for (int64_t t = threadIdx.x; t < tokens; t += 1024) {
    if (!has_loss(targets[t], vocab)) continue;
    const float one = dloss ? dloss[t] : 0.f, all = one + (dlse ? dlse[t] : 0.f);
    top = fmaxf(top, fmaxf(fabsf(one), fabsf(all)));
  }
#pragma unroll
  for (int o = 16; o > 0; o /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = top;
  __syncthreads();
  for (int i = 0; i < 32; ++i) top = fmaxf(top, part[i]);
  // 2^13 over the largest, both rounded down to powers of two; 1 for 0 and infinity
  const int e = (__float_as_int(top) >> 23) - 127;
  const int s = e == -127 || e == 128 ? 0 : (13 - e > 126 ? 126 : (13 - e < -126 ? -126 : 13 - e));
  const float up = __int_as_float((127 + s) << 23), down = __int_as_float((127 - s) << 23);
  if (threadIdx.x == 0) scale[0] = up, scale[1] = down;
  for (int64_t t = threadIdx.x; t < tokens; t += 1024) {
    const int64_t at = targets[t];
    RowCoef q = {0.f, 0.f, 0.f, -1};
    if (has_loss(at, vocab)) {
      const float one = dloss ? dloss[t] : 0.f, all = one + (dlse ? dlse[t] : 0.f);
      q = {all * up, one * up, lse[t] * kLog2e, (int)at};
    }
    rows[t] = q;
  }
}

// Rows into 16-byte aligned ones, padded with zeros to `ld`; rows without a loss
// (where targets are given) become zero.
template <class T>
__global__ void __launch_bounds__(256)
copy_rows_kernel(const T* __restrict__ in, int64_t in_ld, int64_t width, T* __restrict__ out,
                 int64_t ld, int64_t rows, const int64_t* __restrict__ targets, int64_t vocab) {
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const bool keep = targets == nullptr || has_loss(targets[r], vocab);
    for (int64_t c = threadIdx.x; c < ld; c += 256)
      out[r * ld + c] = keep && c < width ? in[r * in_ld + c] : from_f<T>(0.f);
  }
}

template <class T>
__global__ void __launch_bounds__(256)
finish_dx_kernel(const float* __restrict__ sums, int splits, int64_t ld, int64_t tokens,
                 int64_t width, const RowCoef* __restrict__ rows, const float* __restrict__ scale,
                 T* __restrict__ dx, int64_t dx_ld) {
  const float inv = scale[1];
  for (int64_t r = blockIdx.x; r < tokens; r += gridDim.x) {
    const bool keep = rows[r].target >= 0;
    for (int64_t c = threadIdx.x; c < width; c += 256) {
      float v = 0.f;
      for (int s = 0; s < splits; ++s) v += sums[((int64_t)s * tokens + r) * ld + c];
      dx[r * dx_ld + c] = from_f<T>(keep ? v * inv : 0.f);
    }
  }
}

// ---------------------------------------------------------------- host
int pair_count() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    sms = 148;
  return sms / 2;
}

template <class T, int KIND>
ferrum_status run(const CUtensorMap& a, const CUtensorMap& b, Product p, int64_t depth, int splits,
                  cudaStream_t stream, const char* what) {
  static std::atomic<uint64_t> smem_done{0};
  auto kernel = loss_product_kernel<T, KIND>;
  cudaError_t e = launch_detail::ensure_smem(kernel, kSmemBytes, smem_done);
  if (e != cudaSuccess) return cuda_error(e, what);
  p.tiles_m = (int)ceil_div(p.m, kTile), p.tiles_n = (int)ceil_div(p.n, kTile);
  p.steps = (int)ceil_div(depth, kDepth);
  p.steps_per_split = (int)ceil_div(p.steps, splits);
  p.splits = (int)ceil_div(p.steps, p.steps_per_split);      // no empty one
  const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n * p.splits;
  const int grid = 2 * (int)std::min<int64_t>(tiles, pair_count());
  launch_detail::clear_stale_error();
  kernel<<<grid, kThreads, kSmemBytes, stream>>>(a, b, p);
  return launched(what);
}

// An operand as the products need it: the caller's array, or a copy in 16-byte rows.
template <class T>
struct Matrix {
  const T* p;
  int64_t ld;
};
int64_t padded(int64_t n) { return ceil_div(n, 8) * 8; }

template <class T>
ferrum_status copy_rows(const void* in, int64_t in_ld, int64_t width, int64_t rows, T* out,
                        const int64_t* targets, int64_t vocab, cudaStream_t stream,
                        const char* what) {
  launch_detail::clear_stale_error();
  copy_rows_kernel<T><<<(unsigned)std::min<int64_t>(rows, 148 * 64), 256, 0, stream>>>(
      (const T*)in, in_ld, width, out, padded(width), rows, targets, vocab);
  return launched(what);
}

template <class T>
constexpr bool is_bf16() { return std::is_same<T, __nv_bfloat16>::value; }

template <class T>
ferrum_status fwd(ferrum_device* dev, const ferrum_cross_entropy_args* a, cudaStream_t stream,
                  const char* what) {
  const int64_t n = (int64_t)a->tokens, d = (int64_t)a->width, v = (int64_t)a->vocab;
  const bool copy_x = !mappable(a->x, a->x_stride, d), copy_w = !mappable(a->weight, a->weight_stride, d);
  const int64_t ld = padded(d), tiles = ceil_div(v, kTile);
  const size_t x_bytes = copy_x ? (size_t)(n * ld) * 2 : 0, w_bytes = copy_w ? (size_t)(v * ld) * 2 : 0;
  PoolBuffer ws(dev, x_bytes + w_bytes + (size_t)(tiles * n) * sizeof(RowStat) + (size_t)n * 4, stream);
  if (ws.status() != cudaSuccess) return cuda_error(ws.status(), "workspace");
  uint8_t* at = ws.as<uint8_t>();
  Matrix<T> x = {(const T*)a->x, a->x_stride}, w = {(const T*)a->weight, a->weight_stride};
  if (copy_x) {
    if (ferrum_status s = copy_rows<T>(a->x, a->x_stride, d, n, (T*)at, nullptr, 0, stream, what)) return s;
    x = {(const T*)at, ld}, at += x_bytes;
  }
  if (copy_w) {
    if (ferrum_status s = copy_rows<T>(a->weight, a->weight_stride, d, v, (T*)at, nullptr, 0, stream, what)) return s;
    w = {(const T*)at, ld}, at += w_bytes;
  }
  CUtensorMap ma, mb;
  cudaError_t e = tensor_map(&ma, is_bf16<T>(), x.p, d, n, x.ld, kHalf);
  if (e == cudaSuccess) e = tensor_map(&mb, is_bf16<T>(), w.p, d, v, w.ld, kHalf);
  if (e != cudaSuccess) return cuda_error(e, "tensor map");
  Product p = {};
  p.m = n, p.n = v, p.err_flag = dev->err_flag, p.targets = a->targets;
  p.stats = (RowStat*)at, p.at_target = (float*)(p.stats + tiles * n);
  if (ferrum_status s = run<T, kStats>(ma, mb, p, d, 1, stream, what)) return s;
  finish_loss_kernel<<<(unsigned)ceil_div(n, 32), 256, 0, stream>>>(
      p.stats, (int)tiles, n, v, a->targets, p.at_target, a->loss, a->lse);
  return launched(what);
}

// Words of a piece of the vocabulary: 128 MiB of G, but no fewer than 4096.
int64_t piece_of(int64_t tokens, int64_t vocab) {
  const int64_t n = std::max<int64_t>(((int64_t)1 << 26) / tokens / kTile * kTile, 4096);
  return std::min(n, ceil_div(vocab, 32) * 32);
}

template <class T>
ferrum_status bwd(ferrum_device* dev, const ferrum_cross_entropy_args* a, cudaStream_t stream,
                  const char* what) {
  const int64_t n = (int64_t)a->tokens, d = (int64_t)a->width, v = (int64_t)a->vocab;
  const bool copy_w = !mappable(a->weight, a->weight_stride, d);
  const int64_t ld = padded(d), piece = piece_of(n, v);
  // Few tokens make few tiles of dx: its depth is split so that all pairs work.
  const int64_t dx_tiles = ceil_div(n, kTile) * ceil_div(d, kTile);
  const int splits = (int)std::max<int64_t>(
      1, std::min<int64_t>(pair_count() / dx_tiles, ceil_div(piece, 4 * kDepth)));
  auto round = [](size_t b) { return (b + 255) / 256 * 256; };
  const size_t x_bytes = round((size_t)(n * ld) * 2), w_bytes = copy_w ? round((size_t)(v * ld) * 2) : 0;
  const size_t g_bytes = round((size_t)(n * piece) * 2), dx_bytes = round((size_t)(splits * n * ld) * 4);
  PoolBuffer ws(dev, x_bytes + w_bytes + g_bytes + dx_bytes + (size_t)n * sizeof(RowCoef) + 256, stream);
  if (ws.status() != cudaSuccess) return cuda_error(ws.status(), "workspace");
  uint8_t* at = ws.as<uint8_t>();
  T* x = (T*)at;
  at += x_bytes;
  Matrix<T> w = {(const T*)a->weight, a->weight_stride};
  // rows without a loss as zeros, so that nothing of theirs reaches dW
  if (ferrum_status s = copy_rows<T>(a->x, a->x_stride, d, n, x, a->targets, v, stream, what)) return s;
  if (copy_w) {
    if (ferrum_status s = copy_rows<T>(a->weight, a->weight_stride, d, v, (T*)at, nullptr, 0, stream, what)) return s;
    w = {(const T*)at, ld}, at += w_bytes;
  }
  T* g = (T*)at;
  at += g_bytes;
  float* sums = (float*)at;
  at += dx_bytes;
  float* scale = (float*)at;
  RowCoef* rows = (RowCoef*)(at + 256);
  row_coefs_kernel<<<1, 1024, 0, stream>>>(n, v, a->targets, a->lse, a->dloss, a->dlse, rows, scale);
  if (ferrum_status s = launched(what)) return s;

  int used = 1;
  for (int64_t first = 0; first < v; first += piece) {
    const int64_t words = std::min(piece, v - first);
    const T* wp = w.p + first * w.ld;
    CUtensorMap x_k, w_k, g_k, w_mn, g_mn, x_mn;
    cudaError_t e = tensor_map(&x_k, is_bf16<T>(), x, d, n, ld, kHalf);
    if (e == cudaSuccess) e = tensor_map(&w_k, is_bf16<T>(), wp, d, words, w.ld, kHalf);
    if (e == cudaSuccess) e = tensor_map(&g_k, is_bf16<T>(), g, words, n, piece, kHalf);
    if (e == cudaSuccess) e = tensor_map(&w_mn, is_bf16<T>(), wp, d, words, w.ld, kDepth);
    if (e == cudaSuccess) e = tensor_map(&g_mn, is_bf16<T>(), g, words, n, piece, kDepth);
    if (e == cudaSuccess) e = tensor_map(&x_mn, is_bf16<T>(), x, d, n, ld, kDepth);
    if (e != cudaSuccess) return cuda_error(e, "tensor map");
    Product p = {};
    p.err_flag = dev->err_flag, p.rows = rows, p.scale = scale, p.first = first;
    p.m = n, p.n = words, p.out = g, p.ld = piece;
    if (ferrum_status s = run<T, kGrads>(x_k, w_k, p, d, 1, stream, what)) return s;
    p.n = d, p.out = sums, p.ld = ld, p.add = first > 0;
    if (first == 0) {
      const int steps = (int)ceil_div(words, kDepth);
      used = (int)ceil_div(steps, ceil_div(steps, splits));
    }
    if (ferrum_status s = run<T, kDx>(g_k, w_mn, p, words, used, stream, what)) return s;
    p.m = words, p.out = (T*)a->dweight + first * a->dweight_stride, p.ld = a->dweight_stride;
    if (ferrum_status s = run<T, kDw>(g_mn, x_mn, p, n, 1, stream, what)) return s;
  }
  finish_dx_kernel<T><<<(unsigned)std::min<int64_t>(n, 148 * 64), 256, 0, stream>>>(
      sums, used, ld, n, d, rows, scale, (T*)a->dx, a->dx_stride);
  return launched(what);
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
