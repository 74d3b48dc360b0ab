// ferrum_gpu._sequence: the sequence operators (include/ferrum_seq.h) on torch
// tensors. Checks arguments, allocates outputs on the stream the work runs
// on and calls the C ABI. It is compiled because a decode step's kernel takes
// a few microseconds: the same checks in Python took 20 to 30.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <initializer_list>
#include <optional>
#include <sstream>
#include <string>
#include <utility>
#include <vector>

#include "../../../include/ferrum_seq.h"

namespace py = pybind11;

namespace {

using Tensor = at::Tensor;
using Opt = std::optional<at::Tensor>;
using Shape = std::initializer_list<int64_t>;

[[noreturn]] void bad(const std::string& msg) { throw py::value_error(msg); }

std::string dims(at::IntArrayRef s) {
  std::ostringstream o;
  o << s;
  return o.str();
}
std::string type_name(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return "float32";
    case at::kHalf: return "float16";
    case at::kBFloat16: return "bfloat16";
    default: return c10::toString(t);
  }
}
int dtype_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return FERRUM_F32;
    case at::kHalf: return FERRUM_F16;
    case at::kBFloat16: return FERRUM_BF16;
    default: return -1;
  }
}

const Tensor& required(const Opt& t, const char* what) {
  if (!t || !t->defined()) bad(std::string(what) + " is required");
  if (!t->is_cuda()) bad(std::string(what) + " must be a CUDA tensor (got a CPU tensor)");
  return *t;
}
bool given(const Opt& t) { return t && t->defined(); }

void last_contiguous(const Tensor& t, const char* what) {
  if (t.size(-1) > 1 && t.stride(-1) != 1)
    bad(std::string(what) + ": the last dimension must be contiguous");
}

// An activation of `ndim` dimensions (any number for 0).
const Tensor& activation(const Opt& x, const char* what, int ndim, bool contiguous = true) {
  const Tensor& t = required(x, what);
  if (dtype_of(t) < 0)
    bad(std::string(what) + " must be float32, float16 or bfloat16, got " +
        type_name(t.scalar_type()));
  if (ndim ? t.dim() != ndim : t.dim() < 1)
    bad(std::string(what) + " must have " + (ndim ? std::to_string(ndim) : "at least 1") +
        " dimensions, got shape " + dims(t.sizes()));
  if (contiguous) last_contiguous(t, what);
  return t;
}

void place(const Tensor& t, const Tensor& ref, at::IntArrayRef shape, const char* what) {
  if (t.sizes() != shape)
    bad(std::string(what) + " must have shape " + dims(shape) + ", got " + dims(t.sizes()));
  if (t.device() != ref.device())
    bad(std::string(what) + " is on " + t.device().str() + ", expected " + ref.device().str());
}

// A tensor of ref's type and device with the given shape.
const Tensor& like(const Opt& x, const Tensor& ref, at::IntArrayRef shape, const char* what,
                   bool contiguous = true) {
  const Tensor& t = required(x, what);
  if (t.scalar_type() != ref.scalar_type())
    bad(std::string(what) + " must be " + type_name(ref.scalar_type()) + ", got " +
        type_name(t.scalar_type()));
  place(t, ref, shape, what);
  if (contiguous) last_contiguous(t, what);
  return t;
}

// An optional contiguous parameter; its pointer.
template <class P = float>
P* param(const Opt& x, const Tensor& ref, Shape shape, const char* what,
         at::ScalarType type = at::kFloat) {
  if (!given(x)) return nullptr;
  const Tensor& t = required(x, what);
  if (t.scalar_type() != type)
    bad(std::string(what) + " must be " + type_name(type) + ", got " + type_name(t.scalar_type()));
  place(t, ref, shape, what);
  if (!t.is_contiguous()) bad(std::string(what) + " must be contiguous");
  return (P*)t.data_ptr();
}

// An array the call writes: no two of its elements share memory.
const Tensor& writable(const Tensor& t, const char* what) {
  std::vector<std::pair<int64_t, int64_t>> d;
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1) d.emplace_back(t.stride(i), t.size(i));
  std::sort(d.begin(), d.end());
  int64_t reach = 1;
  for (auto [st, n] : d) {
    if (st < reach) bad(std::string(what) + " must not overlap itself");
    reach += st * (n - 1);
  }
  return t;
}

// Whether two tensors have a byte in common: whether the distance of their
// starts is a sum of their strides' multiples, a's forwards and b's backwards.
// The largest strides are tried first, each multiple only if the rest can still
// make up the difference, which leaves few of them where strides nest, as
// slices of one wider array have them. After kTries the answer is yes.
class Overlap {
 public:
  static bool of(const Tensor& a, const Tensor& b) {
    const int64_t gap = (const char*)b.const_data_ptr() - (const char*)a.const_data_ptr();
    if (gap >= 0 ? gap >= bytes(a) : -gap >= bytes(b)) return false;
    if (a.numel() == 0 || b.numel() == 0) return false;
    Overlap o;
    o.add(a, 1), o.add(b, -1);
    std::sort(o.terms_.begin(), o.terms_.end(),
              [](const Term& x, const Term& y) { return x.stride > y.stride; });
    return o.makes(0, gap);
  }

 private:
  struct Term {
    int64_t stride, lo, hi;
  };
  static constexpr int kTries = 1 << 16;
  static int64_t bytes(const Tensor& t) {    // from its start to its end
    if (t.is_contiguous()) return t.nbytes();
    const auto size = t.sizes(), stride = t.strides();
    int64_t n = 1;
    for (size_t i = 0; i < size.size(); ++i) n += (size[i] - 1) * stride[i];
    return n * (int64_t)t.element_size();
  }
  void add(const Tensor& t, int sign) {
    for (int64_t i = 0; i < t.dim(); ++i)
      add(t.stride(i) * (int64_t)t.element_size(), sign * (t.size(i) - 1));
    add(1, sign * ((int64_t)t.element_size() - 1));
  }
  void add(int64_t stride, int64_t most) {   // multiples from 0 to `most`
    if (stride == 0 || most == 0) return;
    auto at = std::find_if(terms_.begin(), terms_.end(),
                           [&](const Term& x) { return x.stride == stride; });
    if (at == terms_.end()) at = terms_.insert(at, Term{stride, 0, 0});
    (most > 0 ? at->hi : at->lo) += most;
  }
  bool makes(size_t k, int64_t gap) {
    if (++tries_ > kTries) return true;
    if (k == terms_.size()) return gap == 0;
    int64_t lo = 0, hi = 0;                  // what the smaller strides can add
    for (size_t i = k + 1; i < terms_.size(); ++i)
      lo += terms_[i].stride * terms_[i].lo, hi += terms_[i].stride * terms_[i].hi;
    const Term& t = terms_[k];
    auto down = [&](int64_t x) { return x >= 0 ? x / t.stride : -((-x + t.stride - 1) / t.stride); };
    const int64_t last = std::min(t.hi, down(gap - lo));
    for (int64_t m = std::max(t.lo, -down(hi - gap)); m <= last; ++m)
      if (makes(k + 1, gap - m * t.stride)) return true;
    return false;
  }
  c10::SmallVector<Term, 10> terms_;
  int tries_ = 0;
};

// Other tensors of a call, by name.
using Named = std::initializer_list<std::pair<const char*, const Opt*>>;

// `t`, which the call writes, shares no memory with the others: blocks run in
// any order, so one would read what another has already written.
void apart(const Tensor& t, const char* what, Named others) {
  for (const auto& [name, x] : others)
    if (given(*x) && Overlap::of(t, **x))
      bad(std::string(what) + " must not share memory with one of the inputs (" + name + ")");
}

// A step's state, or the array that takes the state after it. That may be the
// state itself: each element is then read and written by one thread.
void apart_states(const Opt& state, const Opt& next, Named others) {
  const bool other = given(next) && next->data_ptr() != state->data_ptr();
  if (other) apart(*next, "next_state", {{"state", &state}});
  apart(other ? *next : *state, other ? "next_state" : "state", others);
}

// (batch, rows, values), or (batch, values) for a single step.
ferrum_rows rows(const Tensor& t) {
  return ferrum_rows{t.data_ptr(), t.stride(0), t.dim() > 2 ? t.stride(1) : 0};
}
ferrum_rows rows_or_none(const Opt& t) { return given(t) ? rows(*t) : ferrum_rows{}; }

// Device handle and stream of a call. While it lives, the stream is current,
// so outputs allocated meanwhile belong to it.
class Call {
 public:
  Call(const Tensor& ref, const py::object& device, const py::object& stream)
      : ref_(ref), ordinal_(ref.device().index()) {
    handle_ = handle(device, ordinal_);
    if (stream.is_none()) {
      stream_ = c10::cuda::getCurrentCUDAStream(ordinal_).stream();
    } else {
      const py::object s = py::hasattr(stream, "cuda_stream") ? stream.attr("cuda_stream") : stream;
      try {
        stream_ = (cudaStream_t)s.cast<uintptr_t>();
      } catch (const py::cast_error&) {
        bad("stream must be a cudaStream_t as int or a torch stream, got " +
            py::str(py::type::of(s).attr("__name__")).cast<std::string>());
      }
      other_ = c10::cuda::getStreamFromExternal(stream_, ordinal_);
      guard_.emplace(*other_);
    }
  }
  Tensor empty(at::IntArrayRef shape, at::ScalarType t) const {
    return at::empty(shape, ref_.options().dtype(t));
  }
  Tensor empty_like(const Tensor& x) const { return at::empty(x.sizes(), ref_.options()); }
  Tensor zeros(at::IntArrayRef shape, at::ScalarType t) const {
    return at::zeros(shape, ref_.options().dtype(t));
  }
  // `used`: every tensor of the caller's that the call reads or writes
  template <class Args>
  void run(ferrum_status (*entry)(ferrum_device*, const Args*, void*), Args& a,
           std::initializer_list<const Opt*> used) const {
    a.struct_size = sizeof(Args);
    ferrum_status s;
    {
      py::gil_scoped_release nogil;
      s = entry(handle_, &a, stream_);
    }
    if (s != FERRUM_OK) py::module_::import("ferrum_gpu.capi").attr("check")(s);
    if (other_)
      for (const Opt* x : used)   // the caching allocator must not reuse them early
        if (given(*x)) (*x)->record_stream(*other_);
  }

 private:
  static ferrum_device* handle(const py::object& device, int ordinal) {
    static ferrum_device* known[64] = {};
    if (device.is_none() && ordinal < 64 && known[ordinal]) return known[ordinal];
    auto* h = (ferrum_device*)py::module_::import("ferrum_gpu.device")
                  .attr("_handle")(device, ordinal).cast<uintptr_t>();
    if (device.is_none() && ordinal < 64) known[ordinal] = h;
    return h;
  }
  const Tensor& ref_;
  int ordinal_;
  ferrum_device* handle_;
  cudaStream_t stream_;
  std::optional<c10::cuda::CUDAStream> other_;
  std::optional<c10::cuda::CUDAStreamGuard> guard_;
};

// The caller's `out`, or a new tensor like x.
Tensor output(const Call& c, const Opt& out, const Tensor& x, Named inputs, bool contiguous = true) {
  if (!given(out)) return c.empty_like(x);
  const Tensor& t = writable(like(out, x, x.sizes(), "out", contiguous), "out");
  apart(t, "out", inputs);
  return t;
}

py::object to_py(const Tensor& t) { return t.defined() ? py::cast(t) : py::none(); }

// ---------------------------------------------------------------- short convolution

ferrum_conv1d_args conv_args(const Tensor& x, const Opt& weight, const Opt& bias,
                             const std::optional<std::string>& act, const Opt& state,
                             const Opt& lengths, const char* state_name) {
  if (act && *act != "silu") bad("activation must be None or 'silu', got '" + *act + "'");
  const bool step = x.dim() == 2;
  const int64_t b = x.size(0), n = step ? 1 : x.size(1), d = x.size(-1);
  const Tensor& w = required(weight, "weight");
  if (w.dim() != 2 || w.size(1) < 1 || w.size(1) > FERRUM_CONV1D_MAX_TAPS)
    bad("weight must be (channels, taps) with 1 to 8 taps, got shape " + dims(w.sizes()));
  const int64_t k = w.size(1);
  ferrum_conv1d_args a = {};
  a.dtype = dtype_of(x), a.taps = (int)k, a.silu = act.has_value();
  a.batch = b, a.length = n, a.channels = d;
  a.weight = param(weight, x, {d, k}, "weight");
  a.bias = param(bias, x, {d}, "bias");
  a.initial_state = param<void>(state, x, {b, k - 1, d}, state_name, x.scalar_type());
  a.lengths = param<int32_t>(lengths, x, {b}, "lengths", at::kInt);
  a.x = rows(x);
  return a;
}

py::object causal_conv1d(const Opt& xo, const Opt& weight, const Opt& bias,
                         const std::optional<std::string>& act, const Opt& state,
                         const Opt& lengths, bool want_state, const Opt& out,
                         const py::object& device, const py::object& stream) {
  const Tensor& x = activation(xo, "x", 3);
  auto a = conv_args(x, weight, bias, act, state, lengths, "initial_state");
  Call c(x, device, stream);
  Tensor y = output(c, out, x, {{"x", &xo}, {"weight", &weight}, {"bias", &bias},
                                {"initial_state", &state}, {"lengths", &lengths}});
  Tensor fin;
  if (want_state) fin = c.empty({x.size(0), a.taps - 1, x.size(2)}, x.scalar_type());
  a.y = rows(y);
  if (want_state) a.final_state = fin.data_ptr();
  c.run(ferrum_causal_conv1d, a, {&xo, &weight, &bias, &state, &lengths, &out});
  if (want_state) return py::make_tuple(y, fin);
  return py::cast(y);
}

py::tuple causal_conv1d_backward(const Opt& dyo, const Opt& xo, const Opt& weight, const Opt& bias,
                                 const std::optional<std::string>& act, const Opt& state,
                                 const Opt& lengths, const Opt& dfinal, const py::object& device,
                                 const py::object& stream) {
  const Tensor& x = activation(xo, "x", 3);
  auto a = conv_args(x, weight, bias, act, state, lengths, "initial_state");
  const Tensor& dy = like(dyo, x, x.sizes(), "dy");
  const int64_t b = x.size(0), d = x.size(2);
  a.dfinal_state = param<void>(dfinal, x, {b, a.taps - 1, d}, "dfinal_state", x.scalar_type());
  Call c(x, device, stream);
  Tensor dx = c.empty_like(x), dw = c.empty({d, a.taps}, at::kFloat), db, ds;
  if (given(bias)) db = c.empty({d}, at::kFloat);
  if (given(state)) ds = c.empty({b, a.taps - 1, d}, x.scalar_type());
  a.dy = rows(dy), a.dx = rows(dx);
  a.dweight = (float*)dw.data_ptr();
  if (db.defined()) a.dbias = (float*)db.data_ptr();
  if (ds.defined()) a.dinitial_state = ds.data_ptr();
  c.run(ferrum_causal_conv1d_bwd, a, {&dyo, &xo, &weight, &bias, &state, &lengths, &dfinal});
  return py::make_tuple(dx, dw, to_py(db), to_py(ds));
}

Tensor causal_conv1d_step(const Opt& xo, const Opt& state, const Opt& weight, const Opt& bias,
                          const std::optional<std::string>& act, const Opt& next, const Opt& out,
                          const py::object& device, const py::object& stream) {
  const Tensor& x = activation(xo, "x", 2);
  required(state, "state");
  auto a = conv_args(x, weight, bias, act, state, std::nullopt, "state");
  a.final_state = given(next) ? param<void>(next, x, {x.size(0), a.taps - 1, x.size(1)},
                                            "next_state", x.scalar_type())
                              : (void*)a.initial_state;
  apart_states(state, next, {{"x", &xo}, {"weight", &weight}, {"bias", &bias}});
  Call c(x, device, stream);
  Tensor y = output(c, out, x, {{"x", &xo}, {"weight", &weight}, {"bias", &bias}, {"state", &state},
                                {"next_state", &next}});
  a.y = rows(y);
  c.run(ferrum_causal_conv1d_step, a, {&xo, &state, &next, &weight, &bias, &out});
  return y;
}

// ---------------------------------------------------------------- scan

struct ScanInputs {
  Opt u, delta, A, B, C, D, z, bias;
  bool softplus;
};

ferrum_scan_args scan_args(const ScanInputs& i, const Tensor& u, const Opt& state,
                           const Opt& lengths, const char* state_name) {
  const bool step = u.dim() == 2;
  const int64_t b = u.size(0), n = step ? 1 : u.size(1), d = u.size(-1), lead = u.dim() - 1;
  const Tensor& delta = like(i.delta, u, u.sizes(), "delta");
  if (given(i.z)) like(i.z, u, u.sizes(), "z");
  const Tensor& A = required(i.A, "A");
  if (A.dim() != 2 || A.size(1) < 1 || A.size(1) > FERRUM_SCAN_MAX_STATES)
    bad("A must be (channels, states) with 1 to 64 states, got shape " + dims(A.sizes()));
  const int64_t ns = A.size(1);
  const Tensor &B = required(i.B, "B"), &C = required(i.C, "C");
  const bool grouped = B.dim() == lead + 2;
  const int64_t groups = grouped ? B.size(lead) : 1;
  if (groups < 1 || d % groups != 0)
    bad("the groups of B must divide channels (" + std::to_string(groups) + ", " +
        std::to_string(d) + ")");
  if (C.dim() != B.dim()) bad("B and C must have the same shape");
  c10::SmallVector<int64_t, 4> shape(u.sizes().begin(), u.sizes().end() - 1);
  if (grouped) shape.push_back(groups);
  shape.push_back(ns);
  like(i.B, u, shape, "B"), like(i.C, u, shape, "C");
  ferrum_scan_args a = {};
  a.dtype = dtype_of(u), a.delta_softplus = i.softplus;
  a.batch = b, a.length = n, a.channels = d, a.states = ns, a.groups = groups;
  a.u = rows(u), a.delta = rows(delta), a.z = rows_or_none(i.z);
  a.B = ferrum_rows{B.data_ptr(), B.stride(0), step ? 0 : B.stride(1)};
  a.C = ferrum_rows{C.data_ptr(), C.stride(0), step ? 0 : C.stride(1)};
  if (grouped) a.B_group_stride = B.stride(lead), a.C_group_stride = C.stride(lead);
  a.A = param(i.A, u, {d, ns}, "A");
  a.D = param(i.D, u, {d}, "D");
  a.delta_bias = param(i.bias, u, {d}, "delta_bias");
  a.initial_state = param(state, u, {b, d, ns}, state_name);
  a.lengths = param<int32_t>(lengths, u, {b}, "lengths", at::kInt);
  return a;
}

int64_t saves(const ferrum_scan_args& a) {
  return ((int64_t)a.length + FERRUM_SCAN_SAVE_STEPS - 1) / FERRUM_SCAN_SAVE_STEPS;
}

py::tuple selective_scan(const Opt& uo, const Opt& delta, const Opt& A, const Opt& B, const Opt& C,
                         const Opt& D, const Opt& z, const Opt& bias, bool softplus,
                         const Opt& state, const Opt& lengths, bool save, const Opt& out,
                         const py::object& device, const py::object& stream) {
  const Tensor& u = activation(uo, "u", 3);
  auto a = scan_args({uo, delta, A, B, C, D, z, bias, softplus}, u, state, lengths, "initial_state");
  Call c(u, device, stream);
  Tensor y = output(c, out, u, {{"u", &uo}, {"delta", &delta}, {"z", &z}, {"B", &B}, {"C", &C},
                                {"A", &A}, {"D", &D}, {"delta_bias", &bias},
                                {"initial_state", &state}, {"lengths", &lengths}});
  const int64_t b = u.size(0), d = u.size(2), ns = (int64_t)a.states;
  Tensor fin = c.empty({b, d, ns}, at::kFloat), saved;
  if (save) saved = c.empty({b, saves(a), d, ns}, at::kFloat);
  a.out = rows(y), a.final_state = (float*)fin.data_ptr();
  if (save) a.saved_states = (float*)saved.data_ptr();
  c.run(ferrum_selective_scan, a, {&uo, &delta, &A, &B, &C, &D, &z, &bias, &state, &lengths, &out});
  return py::make_tuple(y, fin, to_py(saved));
}

py::tuple selective_scan_backward(const Opt& douto, const Opt& uo, const Opt& delta, const Opt& A,
                                  const Opt& B, const Opt& C, const Opt& states, const Opt& D,
                                  const Opt& z, const Opt& bias, bool softplus, const Opt& lengths,
                                  const Opt& dfinal, const py::object& device,
                                  const py::object& stream) {
  const Tensor& u = activation(uo, "u", 3);
  auto a = scan_args({uo, delta, A, B, C, D, z, bias, softplus}, u, std::nullopt, lengths, "");
  const Tensor& dout = like(douto, u, u.sizes(), "dout");
  required(states, "states");
  const int64_t b = u.size(0), d = u.size(2), ns = (int64_t)a.states;
  a.saved_states = param(states, u, {b, saves(a), d, ns}, "states");
  a.dfinal_state = param(dfinal, u, {b, d, ns}, "dfinal_state");
  Call c(u, device, stream);
  Tensor du = c.empty_like(u), dd = c.empty_like(u), dz, dD, dbias;
  if (given(z)) dz = c.empty_like(u);
  Tensor dA = c.empty({d, ns}, at::kFloat), dB = c.empty_like(*B), dC = c.empty_like(*C);
  if (given(D)) dD = c.empty({d}, at::kFloat);
  if (given(bias)) dbias = c.empty({d}, at::kFloat);
  Tensor dinit = c.empty({b, d, ns}, at::kFloat);
  a.dout = rows(dout), a.du = rows(du), a.ddelta = rows(dd);
  if (dz.defined()) a.dz = rows(dz);
  a.dA = (float*)dA.data_ptr(), a.dB = dB.data_ptr(), a.dC = dC.data_ptr();
  if (dD.defined()) a.dD = (float*)dD.data_ptr();
  if (dbias.defined()) a.ddelta_bias = (float*)dbias.data_ptr();
  a.dinitial_state = (float*)dinit.data_ptr();
  c.run(ferrum_selective_scan_bwd, a,
        {&douto, &uo, &delta, &A, &B, &C, &states, &D, &z, &bias, &lengths, &dfinal});
  return py::make_tuple(du, dd, dA, dB, dC, to_py(dD), to_py(dz), to_py(dbias), dinit);
}

Tensor selective_scan_step(const Opt& uo, const Opt& delta, const Opt& A, const Opt& B,
                           const Opt& C, const Opt& state, const Opt& D, const Opt& z,
                           const Opt& bias, bool softplus, const Opt& next, const Opt& out,
                           const py::object& device, const py::object& stream) {
  const Tensor& u = activation(uo, "u", 2);
  required(state, "state");
  auto a = scan_args({uo, delta, A, B, C, D, z, bias, softplus}, u, state, std::nullopt, "state");
  a.final_state = given(next) ? param(next, u, {u.size(0), u.size(1), (int64_t)a.states}, "next_state")
                              : (float*)a.initial_state;
  apart_states(state, next, {{"u", &uo}, {"delta", &delta}, {"z", &z}, {"B", &B}, {"C", &C},
                             {"A", &A}, {"D", &D}, {"delta_bias", &bias}});
  Call c(u, device, stream);
  Tensor y = output(c, out, u, {{"u", &uo}, {"delta", &delta}, {"z", &z}, {"B", &B}, {"C", &C},
                                {"A", &A}, {"D", &D}, {"delta_bias", &bias}, {"state", &state},
                                {"next_state", &next}});
  a.out = rows(y);
  c.run(ferrum_selective_scan_step, a,
        {&uo, &delta, &A, &B, &C, &state, &next, &D, &z, &bias, &out});
  return y;
}

// ---------------------------------------------------------------- norms

// (..., channels) as (rows, channels) with one row stride: rows and stride.
struct Matrix {
  int64_t rows, stride;
};
Matrix matrix(const Tensor& t, const char* what) {
  last_contiguous(t, what);
  const int64_t d = t.size(-1);
  if (t.dim() == 1) return {1, d};
  Matrix m{1, 0};
  bool have = false;
  for (int64_t i = t.dim() - 2; i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (!have) {
      m.stride = t.stride(i), have = true;
    } else if (t.numel() && t.stride(i) != m.stride * m.rows) {
      bad(std::string(what) + ": the leading dimensions must collapse to one stride");
    }
    m.rows *= t.size(i);
  }
  return m;
}

ferrum_norm_args norm_args(const Tensor& ref, at::ScalarType res, const std::string& kind,
                           double eps, const Opt& weight, const Opt& bias, const Opt& scale,
                           int64_t groups, bool inside) {
  ferrum_norm_args a = {};
  if (kind == "rms")
    a.kind = FERRUM_NORM_RMS;
  else if (kind == "layer")
    a.kind = FERRUM_NORM_LAYER;
  else
    bad("kind must be 'rms' or 'layer', got '" + kind + "'");
  if (!(eps >= 0.0)) bad("eps must not be negative, got " + std::to_string(eps));
  const int64_t d = ref.size(-1);
  if (groups < 1 || d % groups != 0)
    bad("groups must divide channels (" + std::to_string(groups) + ", " + std::to_string(d) + ")");
  required(weight, "weight");
  a.dtype = dtype_of(ref);
  a.residual_dtype = res == at::kFloat ? FERRUM_F32 : a.dtype;
  a.gate_inside = inside;
  a.rows = d ? ref.numel() / d : 0, a.channels = d, a.groups = groups, a.eps = (float)eps;
  a.weight = param(weight, ref, {d}, "weight");
  a.bias = param(bias, ref, {d}, "bias");
  a.scale = param(scale, ref, {d}, "scale");
  return a;
}

const Tensor& residual_like(const Opt& x, const Tensor& ref, const char* what) {
  const Tensor& t = required(x, what);
  if (t.scalar_type() != at::kFloat && t.scalar_type() != ref.scalar_type())
    bad(std::string(what) + " must be float32 or " + type_name(ref.scalar_type()) + ", got " +
        type_name(t.scalar_type()));
  place(t, ref, ref.sizes(), what);
  return t;
}

Tensor sums_for(const Call& c, const Opt& p) {
  return given(p) ? c.empty(p->sizes(), at::kFloat) : Tensor();
}
float* ptr(const Tensor& t) { return t.defined() ? (float*)t.data_ptr() : nullptr; }

py::tuple norm_before(const Opt& xo, const Opt& weight, const Opt& bias, const Opt& residual,
                      const Opt& scale, const std::string& kind, double eps,
                      const py::object& device, const py::object& stream) {
  const Tensor& x = activation(xo, "x", 0);
  at::ScalarType rt = x.scalar_type();
  if (given(residual)) rt = residual_like(residual, x, "residual").scalar_type();
  auto a = norm_args(x, rt, kind, eps, weight, bias, scale, 1, false);
  a.x_stride = matrix(x, "x").stride;
  if (given(residual)) {
    a.residual_stride = matrix(*residual, "residual").stride;
    a.residual = residual->data_ptr();
  }
  Call c(x, device, stream);
  Tensor y = c.empty_like(x), r = c.empty(x.sizes(), rt);
  a.x = x.data_ptr(), a.y = y.data_ptr(), a.r = r.data_ptr();
  a.y_stride = a.r_stride = x.size(-1);
  c.run(ferrum_norm_before, a, {&xo, &residual, &weight, &bias, &scale});
  return py::make_tuple(y, r);
}

py::tuple norm_before_backward(const Opt& dyo, const Opt& ro, const Opt& weight, const Opt& bias,
                               const Opt& dr, const Opt& x, const Opt& scale,
                               const std::string& kind, double eps, const py::object& device,
                               const py::object& stream) {
  const Tensor& dy = activation(dyo, "dy", 0);
  const Tensor& r = residual_like(ro, dy, "r");
  auto a = norm_args(dy, r.scalar_type(), kind, eps, weight, bias, scale, 1, false);
  a.dy = dy.data_ptr(), a.dy_stride = matrix(dy, "dy").stride;
  a.r = r.data_ptr(), a.r_stride = matrix(r, "r").stride;
  if (given(dr)) {
    like(dr, r, r.sizes(), "dr");
    a.dr = dr->data_ptr(), a.dr_stride = matrix(*dr, "dr").stride;
  }
  if (given(scale)) {
    like(x, dy, dy.sizes(), "x");
    a.x = x->data_ptr(), a.x_stride = matrix(*x, "x").stride;
  }
  Call c(dy, device, stream);
  Tensor dx = c.empty_like(dy), dres = c.empty(dy.sizes(), r.scalar_type());
  Tensor dw = sums_for(c, weight), db = sums_for(c, bias), ds = sums_for(c, scale);
  a.dx = dx.data_ptr(), a.dresidual = dres.data_ptr();
  a.dx_stride = a.dresidual_stride = dy.size(-1);
  a.dweight = ptr(dw), a.dbias = ptr(db), a.dscale = ptr(ds);
  c.run(ferrum_norm_before_bwd, a, {&dyo, &ro, &dr, &x, &weight, &bias, &scale});
  return py::make_tuple(dx, dres, dw, to_py(db), to_py(ds));
}

Tensor norm_after(const Opt& xo, const Opt& weight, const Opt& bias, const Opt& gate, bool inside,
                  const Opt& residual, const Opt& scale, int64_t groups, const std::string& kind,
                  double eps, const Opt& out, const py::object& device, const py::object& stream) {
  const Tensor& x = activation(xo, "x", 0);
  at::ScalarType rt = x.scalar_type();
  if (given(residual)) rt = residual_like(residual, x, "residual").scalar_type();
  auto a = norm_args(x, rt, kind, eps, weight, bias, scale, groups, inside);
  a.x = x.data_ptr(), a.x_stride = matrix(x, "x").stride;
  if (given(gate)) {
    like(gate, x, x.sizes(), "gate");
    a.gate = gate->data_ptr(), a.gate_stride = matrix(*gate, "gate").stride;
  }
  if (given(residual)) {
    a.residual = residual->data_ptr();
    a.residual_stride = matrix(*residual, "residual").stride;
  }
  Call c(x, device, stream);
  Tensor y = output(c, out, x, {{"x", &xo}, {"gate", &gate}, {"residual", &residual},
                                {"weight", &weight}, {"bias", &bias}, {"scale", &scale}});
  a.y = y.data_ptr(), a.y_stride = matrix(y, "out").stride;
  c.run(ferrum_norm_after, a, {&xo, &gate, &residual, &weight, &bias, &scale, &out});
  return y;
}

py::tuple norm_after_backward(const Opt& douto, const Opt& xo, const Opt& weight, const Opt& bias,
                              const Opt& gate, bool inside, const Opt& scale, int64_t groups,
                              const std::string& kind, double eps, const py::object& device,
                              const py::object& stream) {
  const Tensor& x = activation(xo, "x", 0);
  auto a = norm_args(x, x.scalar_type(), kind, eps, weight, bias, scale, groups, inside);
  const Tensor& dout = like(douto, x, x.sizes(), "dout");
  a.x = x.data_ptr(), a.x_stride = matrix(x, "x").stride;
  a.dy = dout.data_ptr(), a.dy_stride = matrix(dout, "dout").stride;
  if (given(gate)) {
    like(gate, x, x.sizes(), "gate");
    a.gate = gate->data_ptr(), a.gate_stride = matrix(*gate, "gate").stride;
  }
  Call c(x, device, stream);
  Tensor dx = c.empty_like(x), dg;
  if (given(gate)) dg = c.empty_like(x);
  Tensor dw = sums_for(c, weight), db = sums_for(c, bias), ds = sums_for(c, scale);
  a.dx = dx.data_ptr();
  if (dg.defined()) a.dgate = dg.data_ptr();
  a.dx_stride = a.dgate_stride = x.size(-1);
  a.dweight = ptr(dw), a.dbias = ptr(db), a.dscale = ptr(ds);
  c.run(ferrum_norm_after_bwd, a, {&douto, &xo, &gate, &weight, &bias, &scale});
  return py::make_tuple(dx, to_py(dg), dw, to_py(db), to_py(ds));
}

// ---------------------------------------------------------------- long convolution

ferrum_long_conv_args long_args(const Tensor& x, at::IntArrayRef shape, const Opt& kernel,
                                const Opt& skip) {
  const int64_t b = shape[0], d = shape[1], n = shape[2];
  const Tensor& k = required(kernel, "kernel");
  if (k.dim() != 2 || (n > 0 && (k.size(1) < 1 || k.size(1) > n)))
    bad("kernel must be (channels, taps) with 1 to " + std::to_string(n) + " taps, got shape " +
        dims(k.sizes()));
  ferrum_long_conv_args a = {};
  a.dtype = dtype_of(x), a.batch = b, a.channels = d, a.length = n, a.kernel_length = k.size(1);
  a.kernel = param(kernel, x, {d, k.size(1)}, "kernel");
  a.skip = param(skip, x, {d}, "skip");
  return a;
}

Tensor long_conv(const Opt& xo, const Opt& kernel, const Opt& skip, const Opt& out,
                 const py::object& device, const py::object& stream) {
  const Tensor& x = activation(xo, "x", 3, false);
  auto a = long_args(x, x.sizes(), kernel, skip);
  Call c(x, device, stream);
  Tensor y = output(c, out, x, {{"x", &xo}, {"kernel", &kernel}, {"skip", &skip}}, false);
  a.x = rows(x), a.x_step = x.stride(2), a.y = rows(y), a.y_step = y.stride(2);
  c.run(ferrum_long_conv, a, {&xo, &kernel, &skip, &out});
  return y;
}

py::tuple long_conv_backward(const Opt& dyo, const Opt& xo, const Opt& kernel, const Opt& skip,
                             const py::object& device, const py::object& stream) {
  const Tensor& x = activation(xo, "x", 3, false);
  auto a = long_args(x, x.sizes(), kernel, skip);
  const Tensor& dy = like(dyo, x, x.sizes(), "dy", false);
  Call c(x, device, stream);
  Tensor dx = c.empty_like(x), dk, ds;
  const bool empty = x.size(2) == 0;       // the C call has nothing to write then
  dk = empty ? c.zeros(kernel->sizes(), at::kFloat) : c.empty(kernel->sizes(), at::kFloat);
  if (given(skip)) ds = empty ? c.zeros(skip->sizes(), at::kFloat) : c.empty(skip->sizes(), at::kFloat);
  a.x = rows(x), a.x_step = x.stride(2), a.dy = rows(dy), a.dy_step = dy.stride(2);
  a.dx = rows(dx), a.dx_step = 1, a.dkernel = ptr(dk), a.dskip = ptr(ds);
  c.run(ferrum_long_conv_bwd, a, {&dyo, &xo, &kernel, &skip});
  return py::make_tuple(dx, dk, to_py(ds));
}

Tensor long_conv_step(const Opt& xo, const Opt& history, const Opt& positions, const Opt& kernel,
                      const Opt& skip, const Opt& out, const py::object& device,
                      const py::object& stream) {
  const Tensor& x = activation(xo, "x", 2);
  const Tensor& h = required(history, "history");
  if (h.dim() != 3 || h.size(2) < 1)
    bad("history must be (batch, channels, capacity), got " + dims(h.sizes()));
  const int64_t shape[3] = {x.size(0), x.size(1), h.size(2)};
  like(history, x, shape, "history");
  auto a = long_args(x, shape, kernel, skip);
  required(positions, "positions");
  a.positions = param<int32_t>(positions, x, {x.size(0)}, "positions", at::kInt);
  apart(writable(h, "history"), "history", {{"x", &xo}, {"kernel", &kernel}, {"skip", &skip},
                                            {"positions", &positions}});
  Call c(x, device, stream);
  Tensor y = output(c, out, x, {{"x", &xo}, {"history", &history}, {"kernel", &kernel},
                                {"skip", &skip}, {"positions", &positions}});
  a.x = rows(x), a.y = rows(y), a.history = rows(h);
  c.run(ferrum_long_conv_step, a, {&xo, &history, &positions, &kernel, &skip, &out});
  return y;
}

}  // namespace

PYBIND11_MODULE(_sequence, m) {
  m.def("causal_conv1d", &causal_conv1d);
  m.def("causal_conv1d_backward", &causal_conv1d_backward);
  m.def("causal_conv1d_step", &causal_conv1d_step);
  m.def("selective_scan", &selective_scan);
  m.def("selective_scan_backward", &selective_scan_backward);
  m.def("selective_scan_step", &selective_scan_step);
  m.def("norm_before", &norm_before);
  m.def("norm_before_backward", &norm_before_backward);
  m.def("norm_after", &norm_after);
  m.def("norm_after_backward", &norm_after_backward);
  m.def("long_conv", &long_conv);
  m.def("long_conv_backward", &long_conv_backward);
  m.def("long_conv_step", &long_conv_step);
  m.def("_shares_memory", &Overlap::of);
}
