// Gated linear recurrence over (batch, length, channels), one state a channel
// (recurrence.cuh has a step's arithmetic). A thread owns a channel of a
// sequence and walks its steps.
//
// Gradient, with G the gradient of the state:  G_t = dout_t + a_{t+1} G_{t+1}.
// It walks backwards over pieces of 16 steps, whose states it computes again
// from the one the forward saved in front of them.
#include "recurrence.cuh"

namespace ferrum {
namespace seq {
namespace {

constexpr int kThreads = 128;
constexpr int kSave = FERRUM_RECURRENCE_SAVE_STEPS;

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
  int64_t batch, length, channels;
};

__device__ __forceinline__ int64_t valid_length(const int32_t* lengths, int64_t b, int64_t length) {
  if (lengths == nullptr) return length;
  const int64_t n = lengths[b];
  return n < 0 ? 0 : (n > length ? length : n);
}

template <class T>
__global__ void __launch_bounds__(kThreads) recurrence_fwd_kernel(RecArrays<T> p) {
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= p.batch * p.channels) return;
  const int64_t b = i / p.channels, d = i % p.channels;
  const int64_t len = valid_length(p.lengths, b, p.length);
  const int64_t saves = (p.length + kSave - 1) / kSave;
  const float decay = p.decay[d];
  float h = p.initial ? p.initial[i] : 0.f;
  for (int64_t t = 0; t < p.length; ++t) {
    if (p.saved && t % kSave == 0) p.saved[(b * saves + t / kSave) * p.channels + d] = h;
    if (t < len) {
      const Decay a = decay_of(decay, gate_of(to_f(p.rg.at(b, t)[d])).on);
      const float u = gate_of(to_f(p.ig.at(b, t)[d])).on * to_f(p.x.at(b, t)[d]);
      h += fmaf(a.m, h, a.root * u);
    }
    p.out.at(b, t)[d] = from_f<T>(t < len ? h : 0.f);
  }
  if (p.final) p.final[i] = h;
}

template <class T>
__global__ void __launch_bounds__(kThreads) recurrence_bwd_kernel(RecArrays<T> p, float* part) {
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= p.batch * p.channels) return;
  const int64_t b = i / p.channels, d = i % p.channels;
  const int64_t len = valid_length(p.lengths, b, p.length);
  const int64_t saves = (p.length + kSave - 1) / kSave;
  const float decay = p.decay[d];
  float later = p.dfinal ? p.dfinal[i] : 0.f, sum = 0.f;
  for (int64_t t = len; t < p.length; ++t)
    p.dx.at(b, t)[d] = p.dig.at(b, t)[d] = p.drg.at(b, t)[d] = from_f<T>(0.f);
  for (int64_t s = (len + kSave - 1) / kSave - 1; s >= 0; --s) {
    const int64_t t0 = s * kSave;
    const int n = (int)(len - t0 < kSave ? len - t0 : kSave);
    float before[kSave];
    float h = p.saved[(b * saves + s) * p.channels + d];
    for (int j = 0; j < n; ++j) {
      before[j] = h;
      const Decay a = decay_of(decay, gate_of(to_f(p.rg.at(b, t0 + j)[d])).on);
      const float u = gate_of(to_f(p.ig.at(b, t0 + j)[d])).on * to_f(p.x.at(b, t0 + j)[d]);
      h += fmaf(a.m, h, a.root * u);
    }
    for (int j = n - 1; j >= 0; --j) {
      const int64_t t = t0 + j;
      const Gate r = gate_of(to_f(p.rg.at(b, t)[d])), ig = gate_of(to_f(p.ig.at(b, t)[d]));
      const Decay a = decay_of(decay, r.on);
      const float g = to_f(p.dout.at(b, t)[d]) + later;
      const StepGrads q = step_grads(g, before[j], to_f(p.x.at(b, t)[d]), ig, r, a, decay);
      p.dx.at(b, t)[d] = from_f<T>(q.dx);
      p.dig.at(b, t)[d] = from_f<T>(q.dig);
      p.drg.at(b, t)[d] = from_f<T>(q.drg);
      sum += q.ddecay;
      later = fmaf(a.m, g, g);
    }
  }
  part[i] = sum;
  if (p.dinitial) p.dinitial[i] = later;
}

template <class T>
__global__ void __launch_bounds__(kThreads) recurrence_step_kernel(RecArrays<T> p) {
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= p.batch * p.channels) return;
  const int64_t b = i / p.channels, d = i % p.channels;
  const Decay a = decay_of(p.decay[d], gate_of(to_f(p.rg.at(b, 0)[d])).on);
  const float u = gate_of(to_f(p.ig.at(b, 0)[d])).on * to_f(p.x.at(b, 0)[d]);
  const float h0 = p.initial[i];
  const float h = h0 + fmaf(a.m, h0, a.root * u);
  p.out.at(b, 0)[d] = from_f<T>(h);
  p.final[i] = h;
}

template <class T>
RecArrays<T> arrays_of(const ferrum_recurrence_args* a) {
  RecArrays<T> p;
  p.x = rows_of<T>(a->x), p.ig = rows_of<T>(a->input_gate), p.rg = rows_of<T>(a->recurrence_gate);
  p.out = rows_of<T>(a->out), p.dout = rows_of<T>(a->dout), p.dx = rows_of<T>(a->dx);
  p.dig = rows_of<T>(a->dinput_gate), p.drg = rows_of<T>(a->drecurrence_gate);
  p.decay = a->decay, p.initial = a->initial_state, p.final = a->final_state;
  p.lengths = a->lengths, p.saved = a->saved_states, p.dfinal = a->dfinal_state;
  p.dinitial = a->dinitial_state;
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
      launch_detail::clear_stale_error();
      recurrence_fwd_kernel<T><<<(unsigned)ceil_div(n, kThreads), kThreads, 0, (cudaStream_t)stream>>>(
          arrays_of<T>(a));
      return launched(what);
    });
  });
}

ferrum_status ferrum_gated_recurrence_bwd(ferrum_device* dev, const ferrum_recurrence_args* a,
                                          void* stream) {
  const char* what = "gated_recurrence_bwd";
  return guarded(what, [&]() -> ferrum_status {
    if (ferrum_status s = check_recurrence(dev, a, what, true)) return s;
    if (a->channels == 0) return FERRUM_OK;
    const int64_t n = (int64_t)a->batch * (int64_t)a->channels;
    cudaStream_t st = (cudaStream_t)stream;
    DeviceGuard guard(dev->ordinal);
    if (guard.status() != cudaSuccess) return cuda_error(guard.status(), "cudaSetDevice");
    return with_dtype(a->dtype, [&](auto tag) -> ferrum_status {
      using T = decltype(tag);
      PoolBuffer ws(dev, (size_t)n * 4 + 4, st);
      if (ws.status() != cudaSuccess) return cuda_error(ws.status(), "workspace");
      if (n > 0) {
        launch_detail::clear_stale_error();
        recurrence_bwd_kernel<T><<<(unsigned)ceil_div(n, kThreads), kThreads, 0, st>>>(
            arrays_of<T>(a), ws.as<float>());
        if (ferrum_status s = launched(what)) return s;
      }
      cudaError_t e = launch_sum_rows(ws.as<float>(), (int64_t)a->batch, (int64_t)a->channels,
                                      (int64_t)a->channels, a->ddecay, nullptr, st);
      return e == cudaSuccess ? FERRUM_OK : cuda_error(e, what);
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
    return with_dtype(a->dtype, [&](auto tag) {
      using T = decltype(tag);
      launch_detail::clear_stale_error();
      recurrence_step_kernel<T><<<(unsigned)ceil_div(n, kThreads), kThreads, 0,
                                  (cudaStream_t)stream>>>(arrays_of<T>(a));
      return launched(what);
    });
  });
}

}  // extern "C"
