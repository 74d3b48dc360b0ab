// The loss against a vocabulary in float32: the products on the FMA pipe, as the
// tensor cores have no product of that precision, with the same epilogues and order of
// kernels as in 16 bits (cross_entropy_tc.cu).
//
// A block of 256 threads computes a tile of 128 x 128 (or of 64 or 32 rows, where there
// are few tiles or tokens), 8 x 8 a thread, two values of a row at a time
// (fma.rn.f32x2), from steps of 16 that it copies to shared memory through registers a
// step ahead. 64 multiply-adds a thread take 4 reads of 16 bytes: bound by the FMA
// pipe (72 TFLOP/s). The depths of dx, the vocabulary, and of dW, the tokens, are split so
// that there are tiles for all SMs; slabs are added in order. No sum is a chain of more
// than 1024 terms (of one as long as a row is wide where logits are made). 4096 x 1024 x
// 4096: 682 us forward (50 TFLOP/s), 2350 for the gradient (44); 16384 x 64 x 256: its
// gradient 114 us, 1125 with dW's depth in one piece.
#include <algorithm>

#include "cross_entropy.cuh"

namespace ferrum {
namespace seq {
namespace {

constexpr int kTile = 128, kStep = 16, kThreads = 256;
// Depth after which the weights' products put their sums down and begin anew: a sum of n terms
// of either sign, one after the other, is off by about 0.4 sqrt(n / 2) units of 2^-24 (dW of
// 65536 x 64 x 256: 3.9e-6 in one chain, the plain form 4.1e-7).
constexpr int kChain = 1024;

enum Kind { kStats, kGrads, kWeights };

// One operand: rows by depth, one of them contiguous, 16-byte rows.
struct Operand {
  const float* p;
  int64_t ld, rows;
  bool along;                // its rows of memory run along the depth's steps (MN-major)
};
struct Product {
  Operand a, b;
  int64_t depth, depth_per_split;
  int tiles_m, tiles_n, splits;
  float* out;                // sums: slabs of a.rows rows
  int64_t ld;
  bool sums, load;           // onto those of earlier pieces
  bool live_rows, live_depth;  // of A; the number of tokens with a loss, shared out to the splits
};
struct Work {
  Product p[2];
  int count;
  const int64_t* targets;    // stats
  RowStat* stats;            // (tile of N, token)
  float* at_target;
  int64_t vocab;
  LiveTokens live;           // gradients
  int64_t first;
};

__device__ __forceinline__ void fma2(float2& d, float2 a, float2 b) {
  uint64_t& r = *(uint64_t*)&d;
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(r) : "l"(*(const uint64_t*)&a), "l"(*(const uint64_t*)&b));
}

// This thread's part of a step's ROWS x 16 values of an operand, on their way to
// shared memory as [depth][row]: units of 4 values.
template <int ROWS>
struct Piece {
  static constexpr int kUnits = ROWS < 64 ? 1 : ROWS / 64, kPitch = ROWS + 4;
  static constexpr int kAcross = ROWS / 4;      // threads across the rows of one step of depth
  const float* p;            // the first unit; the second lies `next` values on
  int64_t next, step;        // and those of the next step of depth `step`
  int rows;                  // of the first unit's row or rows, those that exist
  bool along, second;        // (not along: the second unit's row exists)
  float4 v[kUnits];

  __device__ __forceinline__ Piece(const Operand& o, int64_t r0, int64_t k0) : along(o.along) {
    const int t = threadIdx.x;
    if (along) {
      const int64_t r = r0 + t % kAcross * 4;
      p = o.p + (k0 + t / kAcross) * o.ld + r, next = kThreads / kAcross * o.ld, step = kStep * o.ld;
      rows = (int)(o.rows - r < 4 ? o.rows - r : 4), second = true;
    } else {                 // 4 threads a row
      const int64_t r = r0 + t / 4;
      p = o.p + r * o.ld + k0 + t % 4 * 4, next = 64 * o.ld, step = kStep;
      rows = r < o.rows ? 4 : 0, second = r + 64 < o.rows;
    }
    if (ROWS < 64 && t >= ROWS * 4) rows = 0;
  }
  // The next step, `left` of whose steps of depth exist.
  __device__ __forceinline__ void load(int left) {
    const int t = threadIdx.x;
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      int n;
      if (along)
        n = t / kAcross + kThreads / kAcross * i < left ? rows : 0;
      else
        n = (i == 0 ? rows > 0 : second) ? left - t % 4 * 4 : 0;
      const float* q = p + i * next;
      v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (n >= 4) {
        v[i] = *(const float4*)q;
      } else {
        if (n > 0) v[i].x = q[0];
        if (n > 1) v[i].y = q[1];
        if (n > 2) v[i].z = q[2];
      }
    }
    p += step;
  }
  __device__ __forceinline__ void store(float (*s)[kPitch]) const {
    const int t = threadIdx.x;
    if (ROWS < 64 && t >= ROWS * 4) return;
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      if (along) {
        *(float4*)&s[t / kAcross + kThreads / kAcross * i][t % kAcross * 4] = v[i];
      } else {
        const int r = t / 4 + 64 * i, k = t % 4 * 4;
        s[k][r] = v[i].x, s[k + 1][r] = v[i].y, s[k + 2][r] = v[i].z, s[k + 3][r] = v[i].w;
      }
    }
  }
};

template <int KIND, int ROWS>
__global__ void __launch_bounds__(kThreads, 2) loss_f32_kernel(const __grid_constant__ Work w) {
  constexpr int kMine = ROWS / 16;        // rows of a thread
  __shared__ __align__(16) float sa[2][kStep][ROWS + 4], sb[2][kStep][kTile + 4];
  start_next(), await_previous();
  int t = blockIdx.x;
  const int first = w.p[0].tiles_m * w.p[0].tiles_n * w.p[0].splits;
  const bool second = KIND == kWeights && t >= first;
  if (second) t -= first;
  const Product& p = w.p[second];
  const int split = t / (p.tiles_m * p.tiles_n);
  t %= p.tiles_m * p.tiles_n;
  const int64_t m0 = (int64_t)(t % p.tiles_m) * ROWS, n0 = (int64_t)(t / p.tiles_m) * kTile;
  const int live = KIND == kStats ? 0 : *w.live.count;
  Operand oa = p.a;
  if (p.live_rows) oa.rows = live;
  if (m0 >= oa.rows) return;
  const int64_t each = p.live_depth ? live_each(live, p.splits, kStep) : p.depth_per_split;
  const int64_t k0 = split * each, left = (p.live_depth ? live : p.depth) - k0;
  const int depth = (int)(left < each ? left : each);
  if (depth <= 0) return;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  float2 acc[kMine][4];
#pragma unroll
  for (int i = 0; i < kMine; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = make_float2(0.f, 0.f);
  Piece<ROWS> a(oa, m0, k0);
  Piece<kTile> b(p.b, n0, k0);
  a.load(depth), b.load(depth);
  a.store(sa[0]), b.store(sb[0]);
  __syncthreads();
  int buf = 0, k = kStep, done = 0;
  do {                       // (a chain of sums; one alone but in kWeights)
    const int stop = KIND != kWeights || depth - done <= kChain ? depth : done + kChain;
#pragma unroll 1
    for (; k < stop + kStep; k += kStep, buf ^= 1) {
      const bool more = k < depth;
      if (more) a.load(depth - k), b.load(depth - k);
#pragma unroll
      for (int q = 0; q < kStep; ++q) {
        float x[kMine];
        float2 y[4];
        if constexpr (kMine == 2) {
          *(float2*)&x[0] = *(const float2*)&sa[buf][q][ty * 2];
        } else {
          *(float4*)&x[0] = *(const float4*)&sa[buf][q][ty * 4];
          if constexpr (kMine == 8) *(float4*)&x[4] = *(const float4*)&sa[buf][q][64 + ty * 4];
        }
        *(float4*)&y[0] = *(const float4*)&sb[buf][q][tx * 4];
        *(float4*)&y[2] = *(const float4*)&sb[buf][q][64 + tx * 4];
#pragma unroll
        for (int i = 0; i < kMine; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) fma2(acc[i][j], make_float2(x[i], x[i]), y[j]);
      }
      if (more) a.store(sa[buf ^ 1]), b.store(sb[buf ^ 1]);
      __syncthreads();
    }
    // of a row's values, j < 4 are columns n0 + tx * 4 + j, the others 64 further
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int64_t m = m0 + (kMine == 2 ? ty * 2 + i : i / 4 * 64 + ty * 4 + i % 4);
      const bool row = m < oa.rows;
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = j % 2 ? acc[i][j / 2].y : acc[i][j / 2].x;
      auto column = [&](int j) { return n0 + j / 4 * 64 + tx * 4 + j % 4; };
      if constexpr (KIND == kStats) {
        const int64_t target = row ? w.targets[m] : -1;
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (column(j) >= p.b.rows) v[j] = -INFINITY;
          else if (column(j) == target) w.at_target[m] = v[j];
          top = fmaxf(top, v[j]);
        }
#pragma unroll
        for (int o = 8; o > 0; o /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float shift = shift_of(top), shift2 = shift * kLog2e;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          sum += ex2(fabsf(shift) > kFar ? (v[j] - shift) * kLog2e : fmaf(v[j], kLog2e, -shift2));
#pragma unroll
        for (int o = 8; o > 0; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (row && tx == 0) w.stats[n0 / kTile * p.a.rows + m] = {top, sum};
        continue;
      }
      if (!row) continue;
      float* out = p.out + (p.sums ? split * p.a.rows : 0) * p.ld + m * p.ld;
      if constexpr (KIND == kGrads) {
        const RowCoef q = w.live.rows[m];
        const int64_t at = (int64_t)q.target - w.first;
        const float scale = softmax_scale(q.lse), lse = q.lse * scale;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float g = ex2(fmaf(v[j], scale, -lse)) * q.all - (column(j) == at ? q.one : 0.f);
          v[j] = q.target < 0 ? 0.f : g;
        }
      } else {
        const bool load = p.load || done > 0;
        const float inv = p.sums || stop < depth ? 1.f : w.live.scale[1];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (load && column(j) < p.b.rows) v[j] += out[column(j)];
          v[j] *= inv;
        }
      }
      const bool wide = p.ld % 4 == 0 && (uintptr_t)p.out % 16 == 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t n = column(4 * h);
        if (wide && n + 4 <= p.b.rows) {
          *(float4*)(out + n) = make_float4(v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (n + j < p.b.rows) out[n + j] = v[4 * h + j];
        }
      }
    }
    if constexpr (KIND == kWeights) {
#pragma unroll
      for (int i = 0; i < kMine; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = make_float2(0.f, 0.f);
    }
  } while (KIND == kWeights && (done += kChain) < depth);
}

Product product_of(int tile_rows, const Operand& a, const Operand& b, int64_t depth, int splits = 1) {
  Product p = {};
  p.a = a, p.b = b, p.depth = depth;
  p.tiles_m = (int)ceil_div(a.rows, tile_rows), p.tiles_n = (int)ceil_div(b.rows, kTile);
  p.depth_per_split = ceil_div(ceil_div(depth, kStep), splits) * kStep;
  p.splits = (int)ceil_div(depth, p.depth_per_split);
  return p;
}

// Rows of a tile of m x n: fewer where there are few tokens, and where tiles of more
// leave SMs without work (500 x 384 x 5003, tiles of 128 and 64 rows: 85 and 80 us, the
// gradient 225 and 194; 8 x 1024 x 32000, 128 and 32: 203 and 115, 426 and 287).
int rows_of(int64_t m, int64_t n) {
  if (m <= 32) return 32;
  return ceil_div(m, 128) * ceil_div(n, kTile) < 4 * sm_count() ? 64 : 128;
}

template <int KIND>
ferrum_status run(const Work& w, int tile_rows, bool first, cudaStream_t stream, const char* what) {
  int64_t blocks = 0;
  for (int i = 0; i < w.count; ++i) blocks += (int64_t)w.p[i].tiles_m * w.p[i].tiles_n * w.p[i].splits;
  if (blocks > 0x7fffffff) return invalid(what, "too many tiles for one launch");
  if (tile_rows == 32) return start(what, first, loss_f32_kernel<KIND, 32>, blocks, kThreads, 0, stream, w);
  if (tile_rows == 64) return start(what, first, loss_f32_kernel<KIND, 64>, blocks, kThreads, 0, stream, w);
  if constexpr (KIND == kWeights)
    return invalid(what, "no tile of 128 rows");      // (the gradient asks for 64 or 32)
  else
    return start(what, first, loss_f32_kernel<KIND, 128>, blocks, kThreads, 0, stream, w);
}

bool whole_rows(const void* p, int64_t ld, int64_t cols) {
  return aligned(p, 16) && ld % 4 == 0 && ld >= cols;
}

}  // namespace

ferrum_status loss_fwd_f32(ferrum_device* dev, const ferrum_cross_entropy_args* a,
                           cudaStream_t stream, const char* what) {
  const int64_t n = (int64_t)a->tokens, d = (int64_t)a->width, v = (int64_t)a->vocab;
  const bool copy_x = !whole_rows(a->x, a->x_stride, d), copy_w = !whole_rows(a->weight, a->weight_stride, d);
  const int64_t ld = padded(d), parts = ceil_div(v, kTile);
  PoolBuffer ws(dev, (size_t)((copy_x ? n : 0) + (copy_w ? v : 0)) * ld * 4 +
                         (size_t)(parts * n) * sizeof(RowStat) + (size_t)n * 4, stream);
  if (ws.status() != cudaSuccess) return cuda_error(ws.status(), "workspace");
  uint8_t* at = ws.as<uint8_t>();
  Matrix<float> x = {(const float*)a->x, a->x_stride}, wt = {(const float*)a->weight, a->weight_stride};
  if (copy_x) {
    if (ferrum_status s = copied(x, d, n, at, true, stream, what)) return s;
  }
  if (copy_w) {
    if (ferrum_status s = copied(wt, d, v, at, !copy_x, stream, what)) return s;
  }
  Work w = {};
  const int tile = rows_of(n, v);
  w.p[0] = product_of(tile, {x.p, x.ld, n, false}, {wt.p, wt.ld, v, false}, d), w.count = 1;
  w.targets = a->targets, w.vocab = v;
  w.stats = (RowStat*)at, w.at_target = (float*)(w.stats + parts * n);
  if (ferrum_status s = run<kStats>(w, tile, !copy_x && !copy_w, stream, what)) return s;
  return finish_loss(w.stats, (int)parts, w.at_target, a, stream, what);
}

ferrum_status loss_bwd_f32(ferrum_device* dev, const ferrum_cross_entropy_args* a,
                           cudaStream_t stream, const char* what) {
  const int64_t n = (int64_t)a->tokens, d = (int64_t)a->width, v = (int64_t)a->vocab;
  const bool copy_w = !whole_rows(a->weight, a->weight_stride, d);
  // Words of a piece: 256 MiB of G, but no fewer than 4096.
  const int64_t ld = padded(d);
  const int64_t piece = std::min<int64_t>(
      padded(v), std::max<int64_t>(((int64_t)1 << 26) / n / kTile * kTile, 4096));
  // dx: tiles for two blocks an SM, of 256 words at least
  const int g_tile = rows_of(n, std::min(piece, v)), tile = n <= 32 ? 32 : 64;
  const int64_t dx_tiles = ceil_div(n, tile) * ceil_div(d, kTile);
  const int want = (int)std::max<int64_t>(
      1, std::min<int64_t>(2 * sm_count() / dx_tiles, ceil_div(std::min(piece, v), 256)));
  const int splits = product_of(tile, {nullptr, 0, n, false}, {nullptr, 0, d, false}, std::min(piece, v), want).splits;
  const int64_t rows = ceil_div(n, kStep) * kStep;    // room for all tokens
  // dW: the same, of 256 tokens at least
  const int64_t dw_tiles = ceil_div(std::min(piece, v), tile) * ceil_div(d, kTile);
  const int dw_splits = (int)std::max<int64_t>(1, std::min<int64_t>(2 * sm_count() / dw_tiles, ceil_div(n, 256)));
  auto round = [](int64_t b) { return (size_t)((b + 255) / 256 * 256); };
  const size_t x_bytes = round(rows * ld * 4), w_bytes = copy_w ? round(v * ld * 4) : 0;
  const size_t g_bytes = round(rows * piece * 4), sum_bytes = round(splits * rows * ld * 4);
  const size_t dw_bytes = dw_splits > 1 ? round(dw_splits * std::min(piece, v) * ld * 4) : 0;
  const size_t row_bytes = round(rows * sizeof(RowCoef)), index_bytes = round(rows * 4);
  PoolBuffer ws(dev, x_bytes + w_bytes + g_bytes + sum_bytes + dw_bytes + row_bytes + index_bytes + 256, stream);
  if (ws.status() != cudaSuccess) return cuda_error(ws.status(), "workspace");
  uint8_t* at = ws.as<uint8_t>();
  LiveTokens live;
  live.round = kStep, live.x_rows = rows, live.scale = (float*)at, live.count = (int*)(at + 16);
  live.rows = (RowCoef*)(at += 256), live.index = (int*)(at += row_bytes);
  float* x = (float*)(at += index_bytes);
  float* g = (float*)(at += x_bytes);
  float* sums = (float*)(at += g_bytes);
  float* dw_sums = (float*)(at += sum_bytes);
  at += dw_bytes;
  Matrix<float> wt = {(const float*)a->weight, a->weight_stride};
  if (ferrum_status s = start(what, true, prepare_kernel<float>, blocks_to_prepare(n, ld * 4), 1024, 0,
                              stream, (const float*)a->x, a->x_stride, d, x, ld, n, v, a->targets,
                              (const float*)a->lse, a->dloss, a->dlse, live, (float*)a->dx, a->dx_stride))
    return s;
  if (copy_w) {
    if (ferrum_status s = copied(wt, d, v, at, false, stream, what)) return s;
  }
  for (int64_t first = 0; first < v; first += piece) {
    const int64_t words = std::min(piece, v - first);
    const float* wp = wt.p + first * wt.ld;
    Work w = {};
    w.live = live, w.first = first, w.count = 1;
    w.p[0] = product_of(g_tile, {x, ld, rows, false}, {wp, wt.ld, words, false}, d);
    w.p[0].out = g, w.p[0].ld = piece, w.p[0].live_rows = true;
    if (ferrum_status s = run<kGrads>(w, g_tile, false, stream, what)) return s;
    w.p[0] = product_of(tile, {g, piece, rows, false}, {wp, wt.ld, d, true}, words, splits);
    w.p[0].out = sums, w.p[0].ld = ld, w.p[0].sums = w.p[0].live_rows = true,
     w.p[0].load = first > 0;
    w.p[1] = product_of(tile, {g, piece, words, true}, {x, ld, d, true}, rows);
    float* dw = (float*)a->dweight + first * a->dweight_stride;
    w.p[1].out = dw, w.p[1].ld = a->dweight_stride;
    w.p[1].live_depth = true;
    if (dw_splits > 1) w.p[1].splits = dw_splits, w.p[1].out = dw_sums, w.p[1].ld = ld, w.p[1].sums = true;
    w.count = 2;
    if (ferrum_status s = run<kWeights>(w, tile, false, stream, what)) return s;
    if (dw_splits > 1) {
      const int64_t grid = std::min<int64_t>(ceil_div(words * ld / 4, 256), sm_count() * 16);
      if (ferrum_status s = start(what, false, finish_dw_kernel<float>, grid, 256, 0, stream, (const float*)dw_sums,
                                  dw_splits, kStep, ld, words, d, live, dw, a->dweight_stride))
        return s;
    }
  }
  return start(what, false, finish_dx_kernel<float>, std::min<int64_t>(ceil_div(n * ld / 4, 256), sm_count() * 16),
               256, 0, stream, (const float*)sums, splits, ld, rows, d, live, (float*)a->dx, a->dx_stride);
}

}  // namespace seq
}  // namespace ferrum
