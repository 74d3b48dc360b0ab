// The loss against a vocabulary with its products on the FMA pipe: pieces of
// the vocabulary, whose logits live in a workspace until the next piece.
#include <algorithm>

#include "cross_entropy.cuh"

namespace ferrum {
namespace seq {
namespace {

constexpr int kTile = 128, kStep = 16, kThreads = 256;

// One operand of a product: element (row, k) is at p[row * row_stride + k * k_stride].
// With `targets`, k counts tokens, and those without a loss read as zero.
template <class T>
struct Operand {
  const T* p;
  int64_t row_stride, k_stride, rows;
  const int64_t* targets;
  int64_t vocab;
};

// C[m, n] = alpha sum_k A(m, k) B(n, k) (+ C), a tile of 128 x 128 a block,
// 8 x 8 a thread.
template <class TA, class TB, class TC>
__global__ void __launch_bounds__(kThreads)
product_kernel(Operand<TA> A, Operand<TB> B, TC* C, int64_t ldc, int64_t depth, int64_t col_tiles,
               bool add) {
  __shared__ float sa[kStep][kTile + 4], sb[kStep][kTile + 4];
  const int64_t m0 = blockIdx.x / col_tiles * kTile, n0 = blockIdx.x % col_tiles * kTile;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  float acc[8][8] = {};
  auto stage = [&](auto& op, float (*s)[kTile + 4], int64_t r0, int64_t k0) {
#pragma unroll
    for (int j = 0; j < kTile * kStep / kThreads; ++j) {
      const int e = j * kThreads + threadIdx.x;
      // neighbouring threads along the axis that is contiguous
      const int k = op.k_stride == 1 ? e % kStep : e / kTile;
      const int r = op.k_stride == 1 ? e / kStep : e % kTile;
      float v = 0.f;
      if (r0 + r < op.rows && k0 + k < depth &&
          (op.targets == nullptr || has_loss(op.targets[k0 + k], op.vocab)))
        v = to_f(op.p[(r0 + r) * op.row_stride + (k0 + k) * op.k_stride]);
      s[k][r] = v;
    }
  };
  for (int64_t k0 = 0; k0 < depth; k0 += kStep) {
    stage(A, sa, m0, k0);
    stage(B, sb, n0, k0);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kStep; ++k) {
      float a[8], b[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[i] = sa[k][ty * 4 + i], a[4 + i] = sa[k][64 + ty * 4 + i];
        b[i] = sb[k][tx * 4 + i], b[4 + i] = sb[k][64 + tx * 4 + i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t m = m0 + (i / 4) * 64 + ty * 4 + i % 4;
    if (m >= A.rows) continue;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t n = n0 + (j / 4) * 64 + tx * 4 + j % 4;
      if (n >= B.rows) continue;
      TC* c = C + m * ldc + n;
      *c = from_f<TC>(add ? to_f(*c) + acc[i][j] : acc[i][j]);
    }
  }
}

template <class TA, class TB, class TC>
ferrum_status product(const Operand<TA>& A, const Operand<TB>& B, TC* C, int64_t ldc, int64_t depth,
                      bool add, cudaStream_t stream, const char* what) {
  const int64_t cols = ceil_div(B.rows, kTile), blocks = cols * ceil_div(A.rows, kTile);
  if (blocks > 0x7fffffff) return invalid(what, "too many blocks for one launch");
  launch_detail::clear_stale_error();
  product_kernel<<<(unsigned)blocks, kThreads, 0, stream>>>(A, B, C, ldc, depth, cols, add);
  return launched(what);
}

__device__ RowStat block_join(RowStat s) {
  __shared__ RowStat sh[kThreads];
  sh[threadIdx.x] = s;
  __syncthreads();
  for (int o = kThreads / 2; o > 0; o /= 2) {
    if ((int)threadIdx.x < o) sh[threadIdx.x] = join(sh[threadIdx.x], sh[threadIdx.x + o]);
    __syncthreads();
  }
  return sh[0];
}

// A row's statistics, a block a row, joined with those of the pieces before;
// after the last piece its loss.
__global__ void __launch_bounds__(kThreads)
piece_stats_kernel(const float* __restrict__ logits, int64_t n, int64_t first, LossSizes z,
                   const int64_t* __restrict__ targets, RowStat* stats, float* at_target,
                   float* loss, float* lse) {
  const int64_t t = blockIdx.x;
  const float* l = logits + t * n;
  RowStat s = {-INFINITY, 0.f};
  for (int64_t v = threadIdx.x; v < n; v += kThreads)
    s = join(s, {l[v], fabsf(l[v]) == INFINITY ? ex2(l[v]) : 1.f + (l[v] - l[v])});
  s = block_join(s);
  if (threadIdx.x != 0) return;
  const int64_t at = targets[t] - first;
  const bool counts = has_loss(targets[t], z.vocab);
  if (counts && at >= 0 && at < n) at_target[t] = l[at];
  if (first > 0) s = join(stats[t], s);
  stats[t] = s;
  if (first + n == z.vocab) {
    lse[t] = counts ? lse_of(s) : 0.f;
    loss[t] = counts ? lse_of(s) - at_target[t] : 0.f;
  }
}

// The gradient of a piece's logits, in their place.
__global__ void __launch_bounds__(kThreads)
piece_grads_kernel(float* __restrict__ logits, int64_t n, int64_t first, LossSizes z,
                   const int64_t* __restrict__ targets, const float* __restrict__ lse,
                   const float* __restrict__ dloss, const float* __restrict__ dlse) {
  const int64_t t = blockIdx.x, at = targets[t] - first;
  float* l = logits + t * n;
  const bool counts = has_loss(targets[t], z.vocab);
  const float one = dloss ? dloss[t] : 0.f, all = one + (dlse ? dlse[t] : 0.f), norm = lse[t];
  for (int64_t v = threadIdx.x; v < n; v += kThreads)
    l[v] = counts ? expf(l[v] - norm) * all - (v == at ? one : 0.f) : 0.f;
}

// Columns of a piece: 64 MiB of logits, but no fewer than 1024.
int64_t piece_of(const LossSizes& z) {
  const int64_t n = ((int64_t)1 << 24) / std::max<int64_t>(z.tokens, 1) / 128 * 128;
  return std::min(z.vocab, std::max<int64_t>(n, 1024));
}

LossSizes sizes_of(const ferrum_cross_entropy_args* a) {
  return {(int64_t)a->tokens, (int64_t)a->width, (int64_t)a->vocab};
}

template <class T>
ferrum_status fwd(ferrum_device* dev, const ferrum_cross_entropy_args* a, cudaStream_t stream,
                  const char* what) {
  const LossSizes z = sizes_of(a);
  const int64_t piece = piece_of(z);
  PoolBuffer ws(dev, (size_t)(z.tokens * piece) * 4 + (size_t)z.tokens * 12, stream);
  if (ws.status() != cudaSuccess) return cuda_error(ws.status(), "workspace");
  RowStat* stats = ws.as<RowStat>();
  float* at_target = (float*)(stats + z.tokens);
  float* logits = at_target + z.tokens;
  for (int64_t v = 0; v < z.vocab; v += piece) {
    const int64_t n = std::min(piece, z.vocab - v);
    const Operand<T> x = {(const T*)a->x, a->x_stride, 1, z.tokens, nullptr, 0};
    const Operand<T> w = {(const T*)a->weight + v * a->weight_stride, a->weight_stride, 1, n, nullptr, 0};
    if (ferrum_status s = product(x, w, logits, n, z.width, false, stream, what)) return s;
    piece_stats_kernel<<<(unsigned)z.tokens, kThreads, 0, stream>>>(
        logits, n, v, z, a->targets, stats, at_target, a->loss, a->lse);
    if (ferrum_status s = launched(what)) return s;
  }
  return FERRUM_OK;
}

template <class T>
__global__ void __launch_bounds__(kThreads)
round_rows_kernel(const float* __restrict__ in, T* out, int64_t ld, int64_t width) {
  for (int64_t d = threadIdx.x; d < width; d += kThreads)
    out[blockIdx.x * ld + d] = from_f<T>(in[blockIdx.x * width + d]);
}

template <class T>
ferrum_status bwd(ferrum_device* dev, const ferrum_cross_entropy_args* a, cudaStream_t stream,
                  const char* what) {
  const LossSizes z = sizes_of(a);
  const int64_t piece = piece_of(z);
  PoolBuffer ws(dev, (size_t)(z.tokens * (piece + z.width)) * 4, stream);
  if (ws.status() != cudaSuccess) return cuda_error(ws.status(), "workspace");
  float* logits = ws.as<float>();
  float* sum = logits + z.tokens * piece;
  T* dw = (T*)a->dweight;
  for (int64_t v = 0; v < z.vocab; v += piece) {
    const int64_t n = std::min(piece, z.vocab - v);
    const T* wp = (const T*)a->weight + v * a->weight_stride;
    const Operand<T> x = {(const T*)a->x, a->x_stride, 1, z.tokens, nullptr, 0};
    const Operand<T> w = {wp, a->weight_stride, 1, n, nullptr, 0};
    if (ferrum_status s = product(x, w, logits, n, z.width, false, stream, what)) return s;
    piece_grads_kernel<<<(unsigned)z.tokens, kThreads, 0, stream>>>(
        logits, n, v, z, a->targets, a->lse, a->dloss, a->dlse);
    if (ferrum_status s = launched(what)) return s;
    const Operand<float> g = {logits, n, 1, z.tokens, nullptr, 0};
    const Operand<T> wt = {wp, 1, a->weight_stride, z.width, nullptr, 0};
    if (ferrum_status s = product(g, wt, sum, z.width, n, v > 0, stream, what)) return s;
    const Operand<float> gt = {logits, 1, n, n, nullptr, 0};
    const Operand<T> xt = {(const T*)a->x, 1, a->x_stride, z.width, a->targets, z.vocab};
    if (ferrum_status s = product(gt, xt, dw + v * a->dweight_stride, a->dweight_stride, z.tokens,
                                  false, stream, what))
      return s;
  }
  round_rows_kernel<<<(unsigned)z.tokens, kThreads, 0, stream>>>(sum, (T*)a->dx, a->dx_stride, z.width);
  return launched(what);
}

}  // namespace

ferrum_status loss_fwd_f32(ferrum_device* dev, const ferrum_cross_entropy_args* a,
                           cudaStream_t stream, const char* what) {
  return with_dtype(a->dtype, [&](auto tag) { return fwd<decltype(tag)>(dev, a, stream, what); });
}

ferrum_status loss_bwd_f32(ferrum_device* dev, const ferrum_cross_entropy_args* a,
                           cudaStream_t stream, const char* what) {
  return with_dtype(a->dtype, [&](auto tag) { return bwd<decltype(tag)>(dev, a, stream, what); });
}

}  // namespace seq
}  // namespace ferrum
