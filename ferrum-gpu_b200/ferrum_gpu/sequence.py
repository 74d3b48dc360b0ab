"""Sequence operators on torch CUDA tensors: causal filters and block norms.

What a sequence model runs next to the FFT, without a counterpart in the
reference:

``causal_conv1d``   short depthwise convolution (1 to 8 taps), bias, SiLU
``selective_scan``  input-dependent linear recurrence (state space scan)
``long_conv``       convolution with a filter as long as the sequence, by FFT
``norm_before``     residual update and norm in front of a block
``norm_after``      gated norm behind a block, scaled onto the residual

Each has a ``*_backward``; the filters have a ``*_step`` for one token of
every sequence on kept state. The binding follows ``include/ferrum_seq.h``.

Activations are float32, float16 or bfloat16 tensors, all of one type, shaped
(batch, length, channels) with contiguous channels and any other strides
(``long_conv``: (batch, channels, length), any strides). Parameters, scan
states and parameter gradients are float32. Arithmetic runs in float32; an
output is rounded once to its type. Results do not depend on scheduling.

``lengths`` (int32, one per sequence) are the valid lengths of a padded batch:
steps past them are not read, and their outputs and gradients are zero.

Calls are stream ordered and return without waiting: they run on ``stream``
(a ``cudaStream_t`` as int, or a torch stream), else on torch's current stream
of the tensors' device; outputs belong to that stream. ``device`` is an
optional ``ferrum_gpu.cuda.Device``. Other tensors with a ``__dlpack__``
export on a GPU are taken without a copy.

Errors: ``ValueError`` for arguments, ``ferrum_gpu.capi.FerrumError`` for
failures of the library.
"""

from __future__ import annotations

import contextlib
import ctypes
from typing import NamedTuple, Optional

import torch

from ferrum_gpu import capi
from ferrum_gpu.device import _handle

MAX_TAPS = 8
MAX_STATES = 64
SAVE_STEPS = 16

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_KINDS = {"rms": 0, "layer": 1}

_vp, _i, _sz, _i64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_size_t, ctypes.c_int64


class _Rows(ctypes.Structure):
    _fields_ = [("ptr", _vp), ("batch_stride", _i64), ("row_stride", _i64)]


def _fields(spec: str):
    """Struct fields from "type name name; type name" text."""
    kinds = {"size": _sz, "int": _i, "i64": _i64, "ptr": _vp, "rows": _Rows, "float": ctypes.c_float}
    out = []
    for part in spec.split(";"):
        words = part.split()
        out += [(name, kinds[words[0]]) for name in words[1:]]
    return out


# Mirrors of the argument blocks of include/ferrum_seq.h, field by field.
class ConvArgs(ctypes.Structure):
    _fields_ = _fields("size struct_size; int dtype taps silu; size batch length channels;"
                       "ptr weight bias initial_state lengths; rows x y; ptr final_state;"
                       "rows dy dx; ptr dfinal_state dweight dbias dinitial_state")


class ScanArgs(ctypes.Structure):
    _fields_ = _fields("size struct_size; int dtype delta_softplus;"
                       "size batch length channels states groups; rows u delta z out B C;"
                       "i64 B_group_stride C_group_stride;"
                       "ptr A D delta_bias initial_state final_state lengths saved_states;"
                       "rows dout du ddelta dz; ptr dfinal_state dB dC dA dD ddelta_bias"
                       " dinitial_state")


class NormArgs(ctypes.Structure):
    _fields_ = _fields("size struct_size; int dtype residual_dtype kind gate_inside;"
                       "size rows channels groups; float eps; ptr weight bias scale x gate"
                       " residual y r; i64 x_stride gate_stride residual_stride y_stride r_stride;"
                       "ptr dy dr dx dgate dresidual;"
                       "i64 dy_stride dr_stride dx_stride dgate_stride dresidual_stride;"
                       "ptr dweight dbias dscale")


class LongArgs(ctypes.Structure):
    _fields_ = _fields("size struct_size; int dtype; size batch channels length kernel_length;"
                       "ptr kernel skip; rows x y; i64 x_step y_step; rows dy dx;"
                       "i64 dy_step dx_step; ptr dkernel dskip; rows history; ptr positions")


# entry point -> argument block
SIGNATURES = {
    "ferrum_causal_conv1d": ConvArgs,
    "ferrum_causal_conv1d_bwd": ConvArgs,
    "ferrum_causal_conv1d_step": ConvArgs,
    "ferrum_selective_scan": ScanArgs,
    "ferrum_selective_scan_bwd": ScanArgs,
    "ferrum_selective_scan_step": ScanArgs,
    "ferrum_norm_before": NormArgs,
    "ferrum_norm_before_bwd": NormArgs,
    "ferrum_norm_after": NormArgs,
    "ferrum_norm_after_bwd": NormArgs,
    "ferrum_long_conv": LongArgs,
    "ferrum_long_conv_bwd": LongArgs,
    "ferrum_long_conv_step": LongArgs,
}

_entries: dict = {}


def _entry(name: str):
    fn = _entries.get(name)
    if fn is None:
        fn = getattr(capi.lib(), name)
        fn.restype = _i
        fn.argtypes = [_vp, ctypes.POINTER(SIGNATURES[name]), _vp]
        _entries[name] = fn
    return fn


# ---------------------------------------------------------------- arguments

def _tensor(x, what: str) -> torch.Tensor:
    if not isinstance(x, torch.Tensor):
        dl = getattr(x, "__dlpack_device__", None)
        if dl is None or dl()[0] != 2:   # 2 is kDLCUDA
            raise ValueError(f"{what} must be a CUDA tensor")
        x = torch.from_dlpack(x)
    if not x.is_cuda:
        raise ValueError(f"{what} must be a CUDA tensor (got a CPU tensor)")
    return x


def _activation(x, what: str, ndim: int) -> torch.Tensor:
    x = _tensor(x, what)
    if x.dtype not in _DTYPES:
        raise ValueError(f"{what} must be float32, float16 or bfloat16, got {x.dtype}")
    if x.dim() != ndim:
        raise ValueError(f"{what} must have {ndim} dimensions, got shape {list(x.shape)}")
    return x


def _like(x, ref: torch.Tensor, shape, what: str, contiguous_last: bool = True) -> torch.Tensor:
    """An activation of `ref`'s type and device with the given shape."""
    x = _tensor(x, what)
    if x.dtype != ref.dtype:
        raise ValueError(f"{what} must be {ref.dtype}, got {x.dtype}")
    _place(x, ref, shape, what)
    if contiguous_last and x.shape[-1] > 1 and x.stride(-1) != 1:
        raise ValueError(f"{what}: the last dimension must be contiguous")
    return x


def _place(x: torch.Tensor, ref: torch.Tensor, shape, what: str) -> None:
    if tuple(x.shape) != tuple(shape):
        raise ValueError(f"{what} must have shape {list(shape)}, got {list(x.shape)}")
    if x.device != ref.device:
        raise ValueError(f"{what} is on {x.device}, expected {ref.device}")


def _param(x, ref: torch.Tensor, shape, what: str, dtype=torch.float32) -> Optional[torch.Tensor]:
    """An optional contiguous parameter (float32 unless `dtype` says otherwise)."""
    if x is None:
        return None
    x = _tensor(x, what)
    if x.dtype != dtype:
        raise ValueError(f"{what} must be {dtype}, got {x.dtype}")
    _place(x, ref, shape, what)
    if not x.is_contiguous():
        raise ValueError(f"{what} must be contiguous")
    return x


def _required(x, what: str):
    if x is None:
        raise ValueError(f"{what} is required")
    return x


def _last_contiguous(x: torch.Tensor, what: str) -> torch.Tensor:
    if x.shape[-1] > 1 and x.stride(-1) != 1:
        raise ValueError(f"{what}: the last dimension must be contiguous")
    return x


def _writable(out: torch.Tensor, inputs, what: str = "out") -> torch.Tensor:
    """An output the caller gave: no two of its elements share memory, and it
    starts at none of the inputs."""
    acc = 1
    for st, n in sorted((st, n) for st, n in zip(out.stride(), out.shape) if n > 1):
        if st < acc:
            raise ValueError(f"{what} must not overlap itself")
        acc = st * (n - 1) + acc
    if out.numel() and any(x is not None and x.data_ptr() == out.data_ptr() for x in inputs):
        raise ValueError(f"{what} must not be one of the inputs")
    return out


def _ptr(x: Optional[torch.Tensor]):
    return None if x is None else x.data_ptr()


def _rows(x: Optional[torch.Tensor]) -> _Rows:
    """(batch, rows, values) or, for a single step, (batch, values)."""
    if x is None:
        return _Rows()
    return _Rows(x.data_ptr(), x.stride(0), x.stride(1) if x.dim() > 2 else 0)


class _Call:
    """Device handle and stream of a call; outputs are allocated inside it so
    that they belong to the stream the work runs on."""

    __slots__ = ("handle", "stream", "_scope", "ref")

    def __init__(self, ref: torch.Tensor, device, stream):
        self.ref = ref
        self.handle = _handle(device, ref.device.index)
        if stream is None:
            self.stream = torch.cuda.current_stream(ref.device).cuda_stream
            self._scope = None
        else:
            self.stream = int(getattr(stream, "cuda_stream", stream))
            s = stream if isinstance(stream, torch.cuda.Stream) else torch.cuda.ExternalStream(
                self.stream, device=ref.device)
            self._scope = torch.cuda.stream(s)

    def scope(self):
        return self._scope if self._scope is not None else contextlib.nullcontext()

    def run(self, name: str, args, inputs=()) -> None:
        args.struct_size = ctypes.sizeof(args)
        st = _entry(name)(self.handle, ctypes.byref(args), self.stream)
        if st:
            capi.check(st)
        if self._scope is not None:
            s = self._scope.stream
            for x in inputs:    # the caching allocator must not reuse them early
                if x is not None:
                    x.record_stream(s)


# ---------------------------------------------------------------- short convolution

class ConvGrads(NamedTuple):
    dx: torch.Tensor
    dweight: torch.Tensor
    dbias: Optional[torch.Tensor]
    dinitial_state: Optional[torch.Tensor]


def _conv_common(x, weight, bias, activation, state, lengths, state_name="initial_state"):
    if activation not in (None, "silu"):
        raise ValueError(f"activation must be None or 'silu', got {activation!r}")
    b, n, d = (x.shape[0], 1, x.shape[1]) if x.dim() == 2 else x.shape
    weight = _tensor(_required(weight, "weight"), "weight")
    if weight.dim() != 2 or not 1 <= weight.shape[1] <= MAX_TAPS:
        raise ValueError(f"weight must be (channels, taps) with 1 to {MAX_TAPS} taps, "
                         f"got shape {list(weight.shape)}")
    k = weight.shape[1]
    weight = _param(weight, x, (d, k), "weight")
    bias = _param(bias, x, (d,), "bias")
    state = _param(state, x, (b, k - 1, d), state_name, x.dtype)
    lengths = _param(lengths, x, (b,), "lengths", torch.int32)
    return ConvArgs(dtype=_DTYPES[x.dtype], taps=k, silu=int(activation == "silu"), batch=b,
                    length=n, channels=d, weight=_ptr(weight), bias=_ptr(bias),
                    initial_state=_ptr(state), lengths=_ptr(lengths), x=_rows(x))


def causal_conv1d(x, weight, bias=None, *, activation=None, initial_state=None, lengths=None,
                  return_final_state=False, out=None, device=None, stream=None):
    """y[b,t,d] = act(bias[d] + sum_j weight[d,j] x[b,t-K+1+j,d]).

    x: (batch, length, channels). weight: (channels, taps). initial_state:
    (batch, taps - 1, channels) of x's type, the values in front of x, oldest
    first (zeros without it). Returns y, or (y, final_state) with the state a
    continuation starts from.
    """
    x = _last_contiguous(_activation(x, "x", 3), "x")
    a = _conv_common(x, weight, bias, activation, initial_state, lengths)
    c = _Call(x, device, stream)
    with c.scope():
        if out is None:
            out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        else:
            _writable(_like(out, x, x.shape, "out"), (x, initial_state))
        fin = (torch.empty((a.batch, a.taps - 1, a.channels), dtype=x.dtype, device=x.device)
               if return_final_state else None)
        a.y, a.final_state = _rows(out), _ptr(fin)
        c.run("ferrum_causal_conv1d", a, (x, weight, bias, initial_state, lengths))
    return (out, fin) if return_final_state else out


def causal_conv1d_backward(dy, x, weight, bias=None, *, activation=None, initial_state=None,
                           lengths=None, dfinal_state=None, device=None, stream=None) -> ConvGrads:
    """Gradients of ``causal_conv1d`` for its output's gradient ``dy`` (and
    that of its final state). ``dbias`` and ``dinitial_state`` are None where
    the forward call had no bias or initial state."""
    x = _last_contiguous(_activation(x, "x", 3), "x")
    a = _conv_common(x, weight, bias, activation, initial_state, lengths)
    dy = _like(dy, x, x.shape, "dy")
    dfinal_state = _param(dfinal_state, x, (a.batch, a.taps - 1, a.channels), "dfinal_state",
                          x.dtype)
    c = _Call(x, device, stream)
    with c.scope():
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        dw = torch.empty((a.channels, a.taps), dtype=torch.float32, device=x.device)
        db = torch.empty((a.channels,), dtype=torch.float32, device=x.device) if bias is not None else None
        ds = (torch.empty((a.batch, a.taps - 1, a.channels), dtype=x.dtype, device=x.device)
              if initial_state is not None else None)
        a.dy, a.dx, a.dfinal_state = _rows(dy), _rows(dx), _ptr(dfinal_state)
        a.dweight, a.dbias, a.dinitial_state = _ptr(dw), _ptr(db), _ptr(ds)
        c.run("ferrum_causal_conv1d_bwd", a,
              (dy, x, weight, bias, initial_state, lengths, dfinal_state))
    return ConvGrads(dx, dw, db, ds)


def causal_conv1d_step(x, state, weight, bias=None, *, activation=None, next_state=None,
                       out=None, device=None, stream=None):
    """One step of every sequence. x: (batch, channels); state: (batch,
    taps - 1, channels), updated in place unless ``next_state`` takes the
    state after the step. Returns y (batch, channels)."""
    x = _last_contiguous(_activation(x, "x", 2), "x")
    a = _conv_common(x, weight, bias, activation, _required(state, "state"), None, "state")
    nxt = state if next_state is None else _param(next_state, x, state.shape, "next_state", x.dtype)
    c = _Call(x, device, stream)
    with c.scope():
        if out is None:
            out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        else:
            _writable(_like(out, x, x.shape, "out"), (x, state))
        a.y, a.final_state = _rows(out), _ptr(nxt)
        c.run("ferrum_causal_conv1d_step", a, (x, state, nxt, weight, bias))
    return out


# ---------------------------------------------------------------- scan

class ScanResult(NamedTuple):
    out: torch.Tensor
    final_state: torch.Tensor
    states: Optional[torch.Tensor]


class ScanGrads(NamedTuple):
    du: torch.Tensor
    ddelta: torch.Tensor
    dA: torch.Tensor
    dB: torch.Tensor
    dC: torch.Tensor
    dD: Optional[torch.Tensor]
    dz: Optional[torch.Tensor]
    ddelta_bias: Optional[torch.Tensor]
    dinitial_state: torch.Tensor


def _scan_common(u, delta, A, B, C, D, z, delta_bias, delta_softplus, state, lengths,
                 state_name="initial_state"):
    step = u.dim() == 2
    b, n, d = (u.shape[0], 1, u.shape[1]) if step else u.shape
    delta = _like(delta, u, u.shape, "delta")
    if z is not None:
        z = _like(z, u, u.shape, "z")
    A = _tensor(_required(A, "A"), "A")
    if A.dim() != 2 or not 1 <= A.shape[1] <= MAX_STATES:
        raise ValueError(f"A must be (channels, states) with 1 to {MAX_STATES} states, "
                         f"got shape {list(A.shape)}")
    ns = A.shape[1]
    A = _param(A, u, (d, ns), "A")
    lead = u.dim() - 1
    B, C = _tensor(_required(B, "B"), "B"), _tensor(_required(C, "C"), "C")
    groups = 1
    if B.dim() == lead + 2:
        groups = B.shape[lead]
    if groups < 1 or d % groups:
        raise ValueError(f"the groups of B must divide channels ({groups}, {d})")
    for name, m in (("B", B), ("C", C)):
        shape = tuple(u.shape[:lead]) + ((groups, ns) if m.dim() == lead + 2 else (ns,))
        if m.dim() != B.dim():
            raise ValueError("B and C must have the same shape")
        _like(m, u, shape, name)
    gs = [m.stride(lead) if m.dim() == lead + 2 else 0 for m in (B, C)]
    D = _param(D, u, (d,), "D")
    delta_bias = _param(delta_bias, u, (d,), "delta_bias")
    state = _param(state, u, (b, d, ns), state_name)
    lengths = _param(lengths, u, (b,), "lengths", torch.int32)
    if step:
        bc = [_Rows(m.data_ptr(), m.stride(0), 0) for m in (B, C)]
    else:
        bc = [_Rows(m.data_ptr(), m.stride(0), m.stride(1)) for m in (B, C)]
    return ScanArgs(dtype=_DTYPES[u.dtype], delta_softplus=int(bool(delta_softplus)), batch=b,
                    length=n, channels=d, states=ns, groups=groups, u=_rows(u), delta=_rows(delta),
                    z=_rows(z), B=bc[0], C=bc[1], B_group_stride=gs[0], C_group_stride=gs[1],
                    A=_ptr(A), D=_ptr(D), delta_bias=_ptr(delta_bias), initial_state=_ptr(state),
                    lengths=_ptr(lengths))


def selective_scan(u, delta, A, B, C, *, D=None, z=None, delta_bias=None, delta_softplus=False,
                   initial_state=None, lengths=None, save_states=False, out=None, device=None,
                   stream=None) -> ScanResult:
    """The recurrence, with dt = softplus(delta + delta_bias) or delta + delta_bias:

        h = exp(dt A) h + dt u B,   out = (h . C + D u) * silu(z)

    u, delta, z: (batch, length, channels). A: (channels, states). B, C:
    (batch, length, states) or (batch, length, groups, states); channel d uses
    group d // (channels // groups). initial_state: (batch, channels, states)
    float32. With ``save_states`` the result carries what the backward needs.
    """
    u = _last_contiguous(_activation(u, "u", 3), "u")
    a = _scan_common(u, delta, A, B, C, D, z, delta_bias, delta_softplus, initial_state, lengths)
    c = _Call(u, device, stream)
    with c.scope():
        if out is None:
            out = torch.empty(u.shape, dtype=u.dtype, device=u.device)
        else:
            _writable(_like(out, u, u.shape, "out"), (u, delta, z, B, C))
        fin = torch.empty((a.batch, a.channels, a.states), dtype=torch.float32, device=u.device)
        saved = None
        if save_states:
            saved = torch.empty((a.batch, -(-a.length // SAVE_STEPS), a.channels, a.states),
                                dtype=torch.float32, device=u.device)
        a.out, a.final_state, a.saved_states = _rows(out), _ptr(fin), _ptr(saved)
        c.run("ferrum_selective_scan", a,
              (u, delta, A, B, C, D, z, delta_bias, initial_state, lengths))
    return ScanResult(out, fin, saved)


def selective_scan_backward(dout, u, delta, A, B, C, states, *, D=None, z=None, delta_bias=None,
                            delta_softplus=False, lengths=None, dfinal_state=None, device=None,
                            stream=None) -> ScanGrads:
    """Gradients of ``selective_scan`` for its output's gradient ``dout`` (and
    that of its final state). ``states`` comes from the forward call with
    ``save_states``. ``dD``, ``dz`` and ``ddelta_bias`` are None where the
    forward call lacked the argument."""
    u = _last_contiguous(_activation(u, "u", 3), "u")
    a = _scan_common(u, delta, A, B, C, D, z, delta_bias, delta_softplus, None, lengths)
    dout = _like(dout, u, u.shape, "dout")
    shape = (a.batch, a.channels, a.states)
    states = _param(_required(states, "states"), u,
                    (a.batch, -(-a.length // SAVE_STEPS)) + shape[1:], "states")
    dfinal_state = _param(dfinal_state, u, shape, "dfinal_state")
    c = _Call(u, device, stream)
    with c.scope():
        def new(s, dt=torch.float32):
            return torch.empty(s, dtype=dt, device=u.device)

        du, ddelta = new(u.shape, u.dtype), new(u.shape, u.dtype)
        dz = new(u.shape, u.dtype) if z is not None else None
        dA, dB, dC = new(A.shape), new(B.shape, u.dtype), new(C.shape, u.dtype)
        dD = new((a.channels,)) if D is not None else None
        dbias = new((a.channels,)) if delta_bias is not None else None
        dinit = new(shape)
        a.dout, a.du, a.ddelta, a.dz = _rows(dout), _rows(du), _rows(ddelta), _rows(dz)
        a.saved_states, a.dfinal_state = _ptr(states), _ptr(dfinal_state)
        a.dA, a.dB, a.dC, a.dD = _ptr(dA), _ptr(dB), _ptr(dC), _ptr(dD)
        a.ddelta_bias, a.dinitial_state = _ptr(dbias), _ptr(dinit)
        c.run("ferrum_selective_scan_bwd", a, (dout, u, delta, A, B, C, states, D, z, delta_bias,
                                               lengths, dfinal_state))
    return ScanGrads(du, ddelta, dA, dB, dC, dD, dz, dbias, dinit)


def selective_scan_step(u, delta, A, B, C, state, *, D=None, z=None, delta_bias=None,
                        delta_softplus=False, next_state=None, out=None, device=None, stream=None):
    """One step of every sequence. u, delta, z: (batch, channels); B, C:
    (batch, states) or (batch, groups, states); state: (batch, channels,
    states) float32, updated in place unless ``next_state`` takes the state
    after the step. Returns out (batch, channels)."""
    u = _last_contiguous(_activation(u, "u", 2), "u")
    a = _scan_common(u, delta, A, B, C, D, z, delta_bias, delta_softplus,
                     _required(state, "state"), None, "state")
    nxt = state if next_state is None else _param(next_state, u, state.shape, "next_state")
    c = _Call(u, device, stream)
    with c.scope():
        if out is None:
            out = torch.empty(u.shape, dtype=u.dtype, device=u.device)
        else:
            _writable(_like(out, u, u.shape, "out"), (u, delta, z, B, C))
        a.out, a.final_state = _rows(out), _ptr(nxt)
        c.run("ferrum_selective_scan_step", a, (u, delta, A, B, C, state, nxt, D, z, delta_bias))
    return out


# ---------------------------------------------------------------- norms

class NormBeforeGrads(NamedTuple):
    dx: Optional[torch.Tensor]
    dresidual: torch.Tensor
    dweight: torch.Tensor
    dbias: Optional[torch.Tensor]
    dscale: Optional[torch.Tensor]


class NormAfterGrads(NamedTuple):
    dx: torch.Tensor
    dgate: Optional[torch.Tensor]
    dweight: torch.Tensor
    dbias: Optional[torch.Tensor]
    dscale: Optional[torch.Tensor]


def _matrix(x, what: str) -> torch.Tensor:
    """(..., channels) as (rows, channels) with one row stride, without a copy."""
    if x.dim() < 1:
        raise ValueError(f"{what} must have at least one dimension")
    if x.dim() != 2:
        try:
            x = x.view(-1, x.shape[-1]) if x.numel() else x.reshape(0, x.shape[-1])
        except RuntimeError:
            raise ValueError(f"{what}: the leading dimensions must collapse to one stride") from None
    return _last_contiguous(x, what)


def _norm_args(ref, res_dtype, kind, eps, weight, bias, scale, groups=1, inside=False):
    if kind not in _KINDS:
        raise ValueError(f"kind must be 'rms' or 'layer', got {kind!r}")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    m, d = ref.shape
    if groups < 1 or d % groups:
        raise ValueError(f"groups must divide channels ({groups}, {d})")
    weight = _param(_required(weight, "weight"), ref, (d,), "weight")
    bias, scale = _param(bias, ref, (d,), "bias"), _param(scale, ref, (d,), "scale")
    return NormArgs(residual_dtype=_DTYPES[res_dtype], kind=_KINDS[kind],
                    gate_inside=int(bool(inside)), rows=m, channels=d, groups=groups, eps=eps,
                    weight=_ptr(weight), bias=_ptr(bias), scale=_ptr(scale))


def _row_stride(x: torch.Tensor) -> int:
    return x.stride(0)


def _residual(x, ref_dtype, what):
    x = _tensor(x, what)
    if x.dtype not in (torch.float32, ref_dtype):
        raise ValueError(f"{what} must be float32 or {ref_dtype}, got {x.dtype}")
    return x


def norm_before(x, weight, bias=None, *, residual=None, scale=None, kind="rms", eps=1e-6,
                device=None, stream=None):
    """r = residual + scale * x;  y = N(r) * weight + bias.  Returns (y, r).

    x: (..., channels); residual: same shape, float32 or x's type, which r
    takes over (x's type without a residual); scale: (channels). N is
    v / sqrt(mean(v^2) + eps) ("rms") or (v - mean) / sqrt(var + eps)
    ("layer"). y has x's type.
    """
    x = _tensor(x, "x")
    if x.dtype not in _DTYPES:
        raise ValueError(f"x must be float32, float16 or bfloat16, got {x.dtype}")
    xm = _matrix(x, "x")
    rm, rdt = None, x.dtype
    if residual is not None:
        residual = _residual(residual, x.dtype, "residual")
        _place(residual, x, x.shape, "residual")
        rm, rdt = _matrix(residual, "residual"), residual.dtype
    a = _norm_args(xm, rdt, kind, eps, weight, bias, scale)
    a.dtype = _DTYPES[x.dtype]
    c = _Call(x, device, stream)
    with c.scope():
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        r = torch.empty(x.shape, dtype=rdt, device=x.device)
        d = xm.shape[1]
        a.x, a.x_stride, a.y, a.y_stride, a.r, a.r_stride = (
            _ptr(xm), _row_stride(xm), _ptr(y), d, _ptr(r), d)
        if rm is not None:
            a.residual, a.residual_stride = _ptr(rm), _row_stride(rm)
        c.run("ferrum_norm_before", a, (x, residual, weight, bias, scale))
    return y, r


def norm_before_backward(dy, r, weight, bias=None, *, dr=None, x=None, scale=None, kind="rms",
                         eps=1e-6, device=None, stream=None) -> NormBeforeGrads:
    """Gradients of ``norm_before`` for those of y (``dy``) and of r (``dr``,
    of r's type). ``r`` is the forward's; ``x`` is needed with ``scale``, for
    ``dscale``. ``dresidual`` has r's type, ``dx`` that of dy."""
    dy = _tensor(dy, "dy")
    if dy.dtype not in _DTYPES:
        raise ValueError(f"dy must be float32, float16 or bfloat16, got {dy.dtype}")
    r = _residual(r, dy.dtype, "r")
    _place(r, dy, dy.shape, "r")
    dym, rm = _matrix(dy, "dy"), _matrix(r, "r")
    a = _norm_args(dym, r.dtype, kind, eps, weight, bias, scale)
    a.dtype = _DTYPES[dy.dtype]
    drm = xm = None
    if dr is not None:
        drm = _matrix(_like(dr, r, r.shape, "dr"), "dr")
    if scale is not None:
        xm = _matrix(_like(_required(x, "x"), dy, dy.shape, "x"), "x")
    c = _Call(dy, device, stream)
    with c.scope():
        d = dym.shape[1]
        dx = torch.empty(dy.shape, dtype=dy.dtype, device=dy.device)
        dres = torch.empty(dy.shape, dtype=r.dtype, device=dy.device)
        dw, db, ds = (torch.empty((d,), dtype=torch.float32, device=dy.device) if p is not None
                      else None for p in (weight, bias, scale))
        a.dy, a.dy_stride, a.r, a.r_stride = _ptr(dym), _row_stride(dym), _ptr(rm), _row_stride(rm)
        a.dx, a.dx_stride, a.dresidual, a.dresidual_stride = _ptr(dx), d, _ptr(dres), d
        if drm is not None:
            a.dr, a.dr_stride = _ptr(drm), _row_stride(drm)
        if xm is not None:
            a.x, a.x_stride = _ptr(xm), _row_stride(xm)
        a.dweight, a.dbias, a.dscale = _ptr(dw), _ptr(db), _ptr(ds)
        c.run("ferrum_norm_before_bwd", a, (dy, r, dr, x, weight, bias, scale))
    return NormBeforeGrads(dx, dres, dw, db, ds)


def norm_after(x, weight, bias=None, *, gate=None, gate_inside=True, residual=None, scale=None,
               groups=1, kind="rms", eps=1e-6, out=None, device=None, stream=None):
    """residual + scale * p, with

        gate_inside:  p = N(x * silu(gate)) * weight + bias
        otherwise:    p = (N(x) * weight + bias) * silu(gate)

    x, gate: (..., channels) of one type; residual: float32 or x's type. N
    (see ``norm_before``) runs over each of ``groups`` equal parts of a row.
    """
    x = _tensor(x, "x")
    if x.dtype not in _DTYPES:
        raise ValueError(f"x must be float32, float16 or bfloat16, got {x.dtype}")
    xm = _matrix(x, "x")
    gm = rm = None
    rdt = x.dtype
    if gate is not None:
        gm = _matrix(_like(gate, x, x.shape, "gate"), "gate")
    if residual is not None:
        residual = _residual(residual, x.dtype, "residual")
        _place(residual, x, x.shape, "residual")
        rm, rdt = _matrix(residual, "residual"), residual.dtype
    a = _norm_args(xm, rdt, kind, eps, weight, bias, scale, groups, gate_inside)
    a.dtype = _DTYPES[x.dtype]
    c = _Call(x, device, stream)
    with c.scope():
        if out is None:
            out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            om = out.view(-1, x.shape[-1]) if out.numel() else out.reshape(0, x.shape[-1])
        else:
            om = _writable(_matrix(_like(out, x, x.shape, "out"), "out"), (x, gate, residual))
        a.x, a.x_stride, a.y, a.y_stride = _ptr(xm), _row_stride(xm), _ptr(om), _row_stride(om)
        if gm is not None:
            a.gate, a.gate_stride = _ptr(gm), _row_stride(gm)
        if rm is not None:
            a.residual, a.residual_stride = _ptr(rm), _row_stride(rm)
        c.run("ferrum_norm_after", a, (x, gate, residual, weight, bias, scale))
    return out


def norm_after_backward(dout, x, weight, bias=None, *, gate=None, gate_inside=True, scale=None,
                        groups=1, kind="rms", eps=1e-6, device=None, stream=None) -> NormAfterGrads:
    """Gradients of ``norm_after`` for its output's gradient ``dout``, which
    is also the gradient of the residual."""
    x = _tensor(x, "x")
    if x.dtype not in _DTYPES:
        raise ValueError(f"x must be float32, float16 or bfloat16, got {x.dtype}")
    xm = _matrix(x, "x")
    dm = _matrix(_like(dout, x, x.shape, "dout"), "dout")
    gm = _matrix(_like(gate, x, x.shape, "gate"), "gate") if gate is not None else None
    a = _norm_args(xm, x.dtype, kind, eps, weight, bias, scale, groups, gate_inside)
    a.dtype = _DTYPES[x.dtype]
    c = _Call(x, device, stream)
    with c.scope():
        d = xm.shape[1]
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        dg = torch.empty(x.shape, dtype=x.dtype, device=x.device) if gate is not None else None
        dw, db, ds = (torch.empty((d,), dtype=torch.float32, device=x.device) if p is not None
                      else None for p in (weight, bias, scale))
        a.x, a.x_stride, a.dy, a.dy_stride = _ptr(xm), _row_stride(xm), _ptr(dm), _row_stride(dm)
        a.dx, a.dx_stride = _ptr(dx), d
        if gm is not None:
            a.gate, a.gate_stride, a.dgate, a.dgate_stride = _ptr(gm), _row_stride(gm), _ptr(dg), d
        a.dweight, a.dbias, a.dscale = _ptr(dw), _ptr(db), _ptr(ds)
        c.run("ferrum_norm_after_bwd", a, (dout, x, gate, weight, bias, scale))
    return NormAfterGrads(dx, dg, dw, db, ds)


# ---------------------------------------------------------------- long convolution

class LongGrads(NamedTuple):
    dx: torch.Tensor
    dkernel: torch.Tensor
    dskip: Optional[torch.Tensor]


def _long_common(x, shape, kernel, skip):
    b, d, n = shape
    kernel = _tensor(_required(kernel, "kernel"), "kernel")
    if kernel.dim() != 2 or not (n == 0 or 1 <= kernel.shape[1] <= n):
        raise ValueError(f"kernel must be (channels, taps) with 1 to {n} taps, "
                         f"got shape {list(kernel.shape)}")
    kernel = _param(kernel, x, (d, kernel.shape[1]), "kernel")
    skip = _param(skip, x, (d,), "skip")
    return LongArgs(dtype=_DTYPES[x.dtype], batch=b, channels=d, length=n,
                    kernel_length=kernel.shape[1], kernel=_ptr(kernel), skip=_ptr(skip))


def long_conv(x, kernel, skip=None, *, out=None, device=None, stream=None):
    """y[b,d,t] = sum_{s<=t} kernel[d,s] x[b,d,t-s] + skip[d] x[b,d,t].

    x: (batch, channels, length), any strides (contiguous length is fastest);
    kernel: (channels, taps), taps up to length; skip: (channels). Long rows go
    through the FFT, so an infinity or NaN reaches its whole row.
    """
    x = _activation(x, "x", 3)
    a = _long_common(x, x.shape, kernel, skip)
    c = _Call(x, device, stream)
    with c.scope():
        if out is None:
            out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        else:
            _writable(_like(out, x, x.shape, "out", False), (x,))
        a.x, a.x_step, a.y, a.y_step = _rows(x), x.stride(2), _rows(out), out.stride(2)
        c.run("ferrum_long_conv", a, (x, kernel, skip))
    return out


def long_conv_backward(dy, x, kernel, skip=None, *, device=None, stream=None) -> LongGrads:
    """Gradients of ``long_conv``; ``dskip`` is None without ``skip``."""
    x = _activation(x, "x", 3)
    a = _long_common(x, x.shape, kernel, skip)
    dy = _like(dy, x, x.shape, "dy", False)
    c = _Call(x, device, stream)
    with c.scope():
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        dk = (torch.empty if x.shape[2] else torch.zeros)(kernel.shape, dtype=torch.float32,
                                                          device=x.device)
        ds = ((torch.empty if x.shape[2] else torch.zeros)(skip.shape, dtype=torch.float32,
                                                           device=x.device)
              if skip is not None else None)
        a.x, a.x_step, a.dy, a.dy_step = _rows(x), x.stride(2), _rows(dy), dy.stride(2)
        a.dx, a.dx_step, a.dkernel, a.dskip = _rows(dx), 1, _ptr(dk), _ptr(ds)
        c.run("ferrum_long_conv_bwd", a, (dy, x, kernel, skip))
    return LongGrads(dx, dk, ds)


def long_conv_step(x, history, positions, kernel, skip=None, *, out=None, device=None, stream=None):
    """One token of every sequence. x: (batch, channels); history: (batch,
    channels, capacity) of x's type, contiguous along the last axis, holding
    the tokens before; positions: (batch) int32, where x goes. Stores x and
    returns y (batch, channels). A position outside the history stores nothing
    and its y is zero."""
    x = _last_contiguous(_activation(x, "x", 2), "x")
    history = _tensor(_required(history, "history"), "history")
    if history.dim() != 3 or history.shape[2] < 1:
        raise ValueError(f"history must be (batch, channels, capacity), got {list(history.shape)}")
    _like(history, x, tuple(x.shape) + (history.shape[2],), "history")
    a = _long_common(x, history.shape, kernel, skip)
    positions = _param(_required(positions, "positions"), x, (x.shape[0],), "positions", torch.int32)
    c = _Call(x, device, stream)
    with c.scope():
        if out is None:
            out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        else:
            _writable(_like(out, x, x.shape, "out"), (x, history))
        a.x, a.y, a.history, a.positions = _rows(x), _rows(out), _rows(history), _ptr(positions)
        c.run("ferrum_long_conv_step", a, (x, history, positions, kernel, skip))
    return out


__all__ = ["causal_conv1d", "causal_conv1d_backward", "causal_conv1d_step", "selective_scan",
           "selective_scan_backward", "selective_scan_step", "norm_before", "norm_before_backward",
           "norm_after", "norm_after_backward", "long_conv", "long_conv_backward",
           "long_conv_step", "ConvGrads", "ScanResult", "ScanGrads", "NormBeforeGrads",
           "NormAfterGrads", "LongGrads"]
