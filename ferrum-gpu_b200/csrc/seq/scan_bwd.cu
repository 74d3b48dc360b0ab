// Gradient of the selective scan. With h the states, a_t = exp(dt_t A) and
// gh_t the gradient of h_t:
//   gh_t = C_t dy_t + a_{t+1} gh_{t+1}
//   dC_t = sum_d dy_t h_t,           dB_t = sum_d gh_t dt_t u_t
//   du_t = D dy_t + dt_t sum_n gh_t B_t
//   ddt_t = sum_n gh_t (A a_t h_{t-1} + u_t B_t),   dA = sum_t gh_t dt_t a_t h_{t-1}
// One thread owns one channel. It walks the saved 64-step pieces from the
// last to the first, recomputes a piece's states from the saved one, then
// walks it backwards. dB and dC are summed over the lanes of a warp and, warp
// by warp through a workspace, over the channels of a group, in fixed order.
#include "scan.cuh"

namespace ferrum {
namespace seq {
namespace {

constexpr int kThreads = 32;

template <class T>
struct ScanGrad {
  Rows<T> dout, du, ddelta, dz;
  const float *dfin, *saved;
  float* dinit;
  float *partBC, *partA;  // (warps, batch, length, 2, N) and (batch, channels, N + 2)
};

template <class T, int N>
__global__ void __launch_bounds__(kThreads)
scan_bwd_kernel(ScanIn<T> in, ScanGrad<T> gr, ScanSizes s, int64_t group_blocks) {
  int64_t q = blockIdx.x;
  const int64_t blk = q % group_blocks;
  q /= group_blocks;
  const int64_t g = q % s.groups, b = q / s.groups;
  const int64_t dl = blk * kThreads + threadIdx.x;
  const bool live = dl < s.per_group;
  const int64_t d = g * s.per_group + (live ? dl : 0);
  const int64_t len = scan_length(in.lengths, b, s.length);
  const int64_t sd = (b * s.channels + d) * s.states;
  float A[N], gh[N], dA[N], hist[kSaveSteps][N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    A[n] = n < s.states ? in.A[d * s.states + n] : 0.f;
    gh[n] = (gr.dfin && n < s.states) ? gr.dfin[sd + n] : 0.f;
    dA[n] = 0.f;
  }
  const float skip = in.D ? in.D[d] : 0.f, bias = in.bias ? in.bias[d] : 0.f;
  float dD = 0.f, dbias = 0.f;
  for (int64_t t = s.length - 1; t >= len; --t)
    if (live) {
      gr.du.at(b, t)[d] = from_f<T>(0.f);
      gr.ddelta.at(b, t)[d] = from_f<T>(0.f);
      if (in.z) gr.dz.at(b, t)[d] = from_f<T>(0.f);
    }
  for (int64_t c = s.saves - 1; c >= 0; --c) {
    const int64_t t0 = c * kSaveSteps;
    const int64_t t1 = t0 + kSaveSteps < len ? t0 + kSaveSteps : len;
    const float* h0 = gr.saved + ((b * s.saves + c) * s.channels + d) * s.states;
    float h[N];
#pragma unroll
    for (int n = 0; n < N; ++n) h[n] = n < s.states ? h0[n] : 0.f;
    for (int64_t t = t0; t < t1; ++t) {
      const float x = to_f(in.u.at(b, t)[d]);
      float dt = to_f(in.delta.at(b, t)[d]) + bias;
      if (s.softplus) dt = softplus_f(dt);
      const T* Bt = in.B.at(b, t) + g * in.B_group;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        hist[t - t0][n] = h[n];
        if (n < s.states) h[n] = fmaf(exp2f(dt * A[n] * kLog2e), h[n], dt * x * to_f(Bt[n]));
      }
    }
    for (int64_t t = t1 - 1; t >= t0; --t) {
      const float x = to_f(in.u.at(b, t)[d]);
      const float raw = to_f(in.delta.at(b, t)[d]) + bias;
      const float dt = s.softplus ? softplus_f(raw) : raw;
      const T* Bt = in.B.at(b, t) + g * in.B_group;
      const T* Ct = in.C.at(b, t) + g * in.C_group;
      float dy = to_f(gr.dout.at(b, t)[d]);
      if (!live) dy = 0.f;
      float y = skip * x;
      if (in.z) {
#pragma unroll
        for (int n = 0; n < N; ++n)
          if (n < s.states) y = fmaf(h[n], to_f(Ct[n]), y);
        const float z = to_f(in.z.at(b, t)[d]), sg = sigmoid_f(z);
        if (live) gr.dz.at(b, t)[d] = from_f<T>(dy * y * sg * (1.f + z * (1.f - sg)));
        dy *= z * sg;
      }
      float gB = 0.f, ddt = 0.f;
      float* pb = gr.partBC + (((blk * s.batch + b) * s.groups + g) * s.length + t) * 2 * s.states;
#pragma unroll
      for (int n = 0; n < N; ++n)
        if (n < s.states) {
          const float Bn = to_f(Bt[n]), Cn = to_f(Ct[n]);
          const float cur = fmaf(Cn, dy, live ? gh[n] : 0.f);
          const float sC = warp_sum(dy * h[n]), sB = warp_sum(cur * dt * x);
          if (threadIdx.x == 0) pb[n] = sB, pb[s.states + n] = sC;
          gB = fmaf(cur, Bn, gB);
          const float prev = hist[t - t0][n];
          const float ga = cur * exp2f(dt * A[n] * kLog2e);
          const float gah = ga * prev;
          ddt = fmaf(gah, A[n], ddt);
          dA[n] = fmaf(gah, dt, dA[n]);
          gh[n] = ga;
          h[n] = prev;
        }
      ddt = fmaf(gB, x, ddt);
      if (s.softplus) ddt *= sigmoid_f(raw);
      dbias += ddt;
      dD = fmaf(dy, x, dD);
      if (live) {
        gr.du.at(b, t)[d] = from_f<T>(fmaf(gB, dt, skip * dy));
        gr.ddelta.at(b, t)[d] = from_f<T>(ddt);
      }
    }
  }
  if (!live) return;
  float* pa = gr.partA + (b * s.channels + d) * (s.states + 2);
#pragma unroll
  for (int n = 0; n < N; ++n)
    if (n < s.states) {
      pa[n] = dA[n];
      if (gr.dinit) gr.dinit[sd + n] = gh[n];
    }
  pa[s.states] = dD;
  pa[s.states + 1] = dbias;
}

// dB and dC (batch, length, groups, N) from the warps' sums, in warp order.
template <class T>
__global__ void sum_bc_kernel(const float* __restrict__ part, T* dB, T* dC,
                              const int32_t* __restrict__ lengths, ScanSizes s, int64_t blocks) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t per = s.batch * s.groups * s.length * 2 * s.states;
  if (i >= per) return;
  const int n = (int)(i % s.states);
  const bool isC = (i / s.states) % 2;
  int64_t q = i / (2 * s.states);
  const int64_t t = q % s.length;
  q /= s.length;
  const int64_t g = q % s.groups, b = q / s.groups;
  float v = 0.f;
  if (t < scan_length(lengths, b, s.length))
    for (int64_t k = 0; k < blocks; ++k) v += part[k * per + i];
  (isC ? dC : dB)[((b * s.length + t) * s.groups + g) * s.states + n] = from_f<T>(v);
}

// dA, dD and the bias gradient: sums over the batch, in order.
__global__ void sum_params_kernel(const float* __restrict__ part, float* dA, float* dD,
                                  float* dbias, ScanSizes s) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t w = s.states + 2, per = s.channels * w;
  if (i >= per) return;
  float v = 0.f;
  for (int64_t b = 0; b < s.batch; ++b) v += part[b * per + i];
  const int64_t d = i / w;
  const int n = (int)(i % w);
  if (n < s.states)
    dA[d * s.states + n] = v;
  else if (n == s.states) {
    if (dD) dD[d] = v;
  } else if (dbias) {
    dbias[d] = v;
  }
}

}  // namespace
}  // namespace seq
}  // namespace ferrum

using namespace ferrum;
using namespace ferrum::seq;

extern "C" ferrum_status ferrum_selective_scan_bwd(ferrum_device* dev, const ferrum_scan_args* a,
                                                   void* stream) {
  const char* what = "selective_scan_bwd";
  return guarded(what, [&]() -> ferrum_status {
    if (ferrum_status s = check_scan(dev, a, what, true)) return s;
    if (a->channels == 0) return FERRUM_OK;
    cudaStream_t st = (cudaStream_t)stream;
    const ScanSizes s = scan_sizes(a);
    const int64_t group_blocks = ceil_div(s.per_group, kThreads);
    const int64_t blocks = s.batch * s.groups * group_blocks;
    const int64_t bc = s.batch * s.groups * s.length * 2 * s.states;
    const int64_t pa = s.channels * (s.states + 2);
    if (blocks > 0x7fffffff || ceil_div(bc, 256) > 0x7fffffff)
      return invalid(what, "too many blocks for one launch");
    DeviceGuard guard(dev->ordinal);
    if (guard.status() != cudaSuccess) return cuda_error(guard.status(), "cudaSetDevice");
    PoolBuffer wbc(dev, (size_t)(group_blocks * bc) * 4 + 4, st);
    PoolBuffer wa(dev, (size_t)(s.batch * pa) * 4 + 4, st);
    if (wbc.status() != cudaSuccess) return cuda_error(wbc.status(), "workspace");
    if (wa.status() != cudaSuccess) return cuda_error(wa.status(), "workspace");
    return with_dtype(a->dtype, [&](auto tag) -> ferrum_status {
      using T = decltype(tag);
      ScanGrad<T> gr{rows_of<T>(a->dout), rows_of<T>(a->du), rows_of<T>(a->ddelta),
                     rows_of<T>(a->dz), a->dfinal_state, a->saved_states, a->dinitial_state,
                     wbc.as<float>(), wa.as<float>()};
      if (blocks > 0) {
        ferrum_status r = with_states(s.states, [&](auto n) {
          launch_detail::clear_stale_error();
          scan_bwd_kernel<T, decltype(n)::value>
              <<<(unsigned)blocks, kThreads, 0, st>>>(scan_in<T>(a), gr, s, group_blocks);
          return launched(what);
        });
        if (r) return r;
      }
      launch_detail::clear_stale_error();
      if (bc > 0)
        sum_bc_kernel<T><<<(unsigned)ceil_div(bc, 256), 256, 0, st>>>(
            wbc.as<float>(), (T*)a->dB, (T*)a->dC, a->lengths, s, group_blocks);
      sum_params_kernel<<<(unsigned)ceil_div(pa, 256), 256, 0, st>>>(wa.as<float>(), a->dA, a->dD,
                                                                    a->ddelta_bias, s);
      return launched(what);
    });
  });
}
