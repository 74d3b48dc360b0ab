// Selective state space scan over (batch, length, channels), forward:
//   dt = softplus(delta + bias),  h[n] = exp(dt A[n]) h[n] + dt u B[n],
//   out = (sum_n h[n] C[n] + D u) * silu(z)
// One thread owns one channel of one sequence and its N states in registers
// and walks the steps; lanes span adjacent channels, so u, delta, z and out
// are read and written in whole segments and B, C are broadcast.
#include "scan.cuh"

namespace ferrum {
namespace seq {
namespace {

constexpr int kThreads = 64;

template <class T, int N>
__global__ void __launch_bounds__(kThreads)
scan_fwd_kernel(ScanIn<T> in, Rows<T> out, float* fin, float* __restrict__ saved, ScanSizes s,
                int64_t col_blocks) {
  const int64_t b = blockIdx.x / col_blocks;
  const int64_t d = (blockIdx.x % col_blocks) * kThreads + threadIdx.x;
  if (d >= s.channels) return;
  const int64_t len = scan_length(in.lengths, b, s.length), g = d / s.per_group;
  const int64_t sd = (b * s.channels + d) * s.states;
  float h[N], a2[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    a2[n] = n < s.states ? in.A[d * s.states + n] * kLog2e : 0.f;
    h[n] = (in.initial && n < s.states) ? in.initial[sd + n] : 0.f;
  }
  const float skip = in.D ? in.D[d] : 0.f, bias = in.bias ? in.bias[d] : 0.f;
  for (int64_t t = 0; t < s.length; ++t) {
    if (saved != nullptr && t % kSaveSteps == 0) {
      float* o = saved + ((b * s.saves + t / kSaveSteps) * s.channels + d) * s.states;
#pragma unroll
      for (int n = 0; n < N; ++n)
        if (n < s.states) o[n] = h[n];
    }
    if (t >= len) {
      out.at(b, t)[d] = from_f<T>(0.f);
      continue;
    }
    const float x = to_f(in.u.at(b, t)[d]);
    float dt = to_f(in.delta.at(b, t)[d]) + bias;
    if (s.softplus) dt = softplus_f(dt);
    const float dx = dt * x;
    const T* Bt = in.B.at(b, t) + g * in.B_group;
    const T* Ct = in.C.at(b, t) + g * in.C_group;
    float y = skip * x;
#pragma unroll
    for (int n = 0; n < N; ++n)
      if (n < s.states) {
        h[n] = fmaf(exp2f(dt * a2[n]), h[n], dx * to_f(Bt[n]));
        y = fmaf(h[n], to_f(Ct[n]), y);
      }
    if (in.z) {
      const float z = to_f(in.z.at(b, t)[d]);
      y *= z * sigmoid_f(z);
    }
    out.at(b, t)[d] = from_f<T>(y);
  }
  if (fin != nullptr)
#pragma unroll
    for (int n = 0; n < N; ++n)
      if (n < s.states) fin[sd + n] = h[n];
}

ferrum_status scan_fwd(ferrum_device* dev, const ferrum_scan_args* a, cudaStream_t stream,
                       const char* what) {
  if (a->batch == 0 || a->channels == 0) return FERRUM_OK;
  const ScanSizes s = scan_sizes(a);
  const int64_t col_blocks = ceil_div(s.channels, kThreads), blocks = s.batch * col_blocks;
  if (blocks > 0x7fffffff) return invalid(what, "too many blocks for one launch");
  DeviceGuard guard(dev->ordinal);
  if (guard.status() != cudaSuccess) return cuda_error(guard.status(), "cudaSetDevice");
  return with_dtype(a->dtype, [&](auto tag) {
    using T = decltype(tag);
    return with_states(s.states, [&](auto n) {
      launch_detail::clear_stale_error();
      scan_fwd_kernel<T, decltype(n)::value><<<(unsigned)blocks, kThreads, 0, stream>>>(
          scan_in<T>(a), rows_of<T>(a->out), a->final_state, a->saved_states, s, col_blocks);
      return launched(what);
    });
  });
}

}  // namespace

ferrum_status check_scan(const ferrum_device* dev, const ferrum_scan_args* a, const char* what,
                         bool bwd) {
  if (ferrum_status s = check_args(dev, a, what)) return s;
  if (a->states < 1 || a->states > FERRUM_SCAN_MAX_STATES)
    return invalid(what, "states must be in [1, 64], got " + std::to_string(a->states));
  if (a->groups < 1 || a->channels % a->groups != 0)
    return invalid(what, "groups must divide channels (" + std::to_string(a->groups) + ", " +
                             std::to_string(a->channels) + ")");
  if (bounded_product({a->batch, a->length + 1, a->channels, a->states}) < 0)
    return invalid(what, "batch * length * channels * states is too large");
  const size_t e = dtype_size(a->dtype);
  const bool none = a->batch == 0 || a->channels == 0, empty = none || a->length == 0;
  if (ferrum_status s = check_ptr(a->A, 4, none, what, "A")) return s;
  if (ferrum_status s = check_ptr(a->D, 4, true, what, "D")) return s;
  if (ferrum_status s = check_ptr(a->delta_bias, 4, true, what, "delta_bias")) return s;
  if (ferrum_status s = check_ptr(a->lengths, 4, true, what, "lengths")) return s;
  if (ferrum_status s = check_ptr(a->initial_state, 4, true, what, "initial_state")) return s;
  if (ferrum_status s = check_ptr(a->u.ptr, e, empty, what, "u")) return s;
  if (ferrum_status s = check_ptr(a->delta.ptr, e, empty, what, "delta")) return s;
  if (ferrum_status s = check_ptr(a->B.ptr, e, empty, what, "B")) return s;
  if (ferrum_status s = check_ptr(a->C.ptr, e, empty, what, "C")) return s;
  if (ferrum_status s = check_ptr(a->z.ptr, e, true, what, "z")) return s;
  if (!bwd) {
    if (ferrum_status s = check_ptr(a->out.ptr, e, empty, what, "out")) return s;
    if (ferrum_status s = check_ptr(a->final_state, 4, true, what, "final_state")) return s;
    return check_ptr(a->saved_states, 4, true, what, "saved_states");
  }
  if (ferrum_status s = check_ptr(a->saved_states, 4, empty, what, "saved_states")) return s;
  if (ferrum_status s = check_ptr(a->dout.ptr, e, empty, what, "dout")) return s;
  if (ferrum_status s = check_ptr(a->du.ptr, e, empty, what, "du")) return s;
  if (ferrum_status s = check_ptr(a->ddelta.ptr, e, empty, what, "ddelta")) return s;
  if (ferrum_status s = check_ptr(a->dz.ptr, e, empty || a->z.ptr == nullptr, what, "dz")) return s;
  if (ferrum_status s = check_ptr(a->dB, e, empty, what, "dB")) return s;
  if (ferrum_status s = check_ptr(a->dC, e, empty, what, "dC")) return s;
  if (ferrum_status s = check_ptr(a->dA, 4, a->channels == 0, what, "dA")) return s;
  if (ferrum_status s = check_ptr(a->dD, 4, true, what, "dD")) return s;
  if (ferrum_status s = check_ptr(a->ddelta_bias, 4, true, what, "ddelta_bias")) return s;
  if (ferrum_status s = check_ptr(a->dfinal_state, 4, true, what, "dfinal_state")) return s;
  return check_ptr(a->dinitial_state, 4, true, what, "dinitial_state");
}

}  // namespace seq
}  // namespace ferrum

using namespace ferrum;
using namespace ferrum::seq;

extern "C" {

ferrum_status ferrum_selective_scan(ferrum_device* dev, const ferrum_scan_args* a, void* stream) {
  const char* what = "selective_scan";
  return guarded(what, [&]() -> ferrum_status {
    if (ferrum_status s = check_scan(dev, a, what, false)) return s;
    return scan_fwd(dev, a, (cudaStream_t)stream, what);
  });
}

ferrum_status ferrum_selective_scan_step(ferrum_device* dev, const ferrum_scan_args* a,
                                         void* stream) {
  const char* what = "selective_scan_step";
  return guarded(what, [&]() -> ferrum_status {
    if (ferrum_status s = check_scan(dev, a, what, false)) return s;
    if (a->length != 1) return invalid(what, "length must be 1, got " + std::to_string(a->length));
    if (a->batch > 0 && a->channels > 0 &&
        (a->initial_state == nullptr || a->final_state == nullptr))
      return invalid(what, "initial_state and final_state are required");
    return scan_fwd(dev, a, (cudaStream_t)stream, what);
  });
}

}  // extern "C"
