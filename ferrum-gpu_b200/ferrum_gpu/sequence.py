"""Sequence operators on torch CUDA tensors: causal filters and block norms.

What a sequence model runs next to the FFT, without a counterpart in the
reference:

``causal_conv1d``   short depthwise convolution (1 to 8 taps), bias, SiLU
``selective_scan``  input-dependent linear recurrence (state space scan)
``long_conv``       convolution with a filter as long as the sequence, by FFT
``norm_before``     residual update and norm in front of a block
``norm_after``      gated norm behind a block, scaled onto the residual

The calls are not recorded by autograd: a result does not require a gradient,
whatever its arguments do. Each operator has a ``*_backward`` instead, to be
called from a ``torch.autograd.Function`` (``examples/sequence_block.py`` has one
for each). The filters have a ``*_step`` for one token of
every sequence on kept state. They call the C ABI of ``include/ferrum_seq.h``
(``ferrum_gpu.capi`` binds it for callers with raw pointers).

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

``out``, ``next_state``, a state updated in place and ``history`` may not share
memory with a call's other tensors (``next_state`` may be ``state``); columns of
one wider array are fine.

Errors: ``ValueError`` for arguments, ``ferrum_gpu.capi.FerrumError`` for
failures of the library.
"""

from __future__ import annotations

import inspect
from typing import NamedTuple, Optional

import torch

from ferrum_gpu import _sequence

MAX_TAPS = 8
MAX_STATES = 64
SAVE_STEPS = 16


def _call(fn, *args):
    """``fn(*args)``, ``args`` ending with the call's stream; tensors of other
    libraries are taken over DLPack."""
    try:
        return fn(*args)
    except TypeError as e:
        _check_types(fn.__name__, args)
        taken = [_from_dlpack(a, args[-1]) for a in args]
        if all(a is b for a, b in zip(taken, args)):
            raise ValueError(str(e).split("\n")[0]) from None
        return fn(*taken)


# Arguments that are no tensors: what they must be, and whether one is.
_OTHERS = {
    "activation": ("None or a string", lambda v: v is None or isinstance(v, str)),
    "kind": ("a string", lambda v: isinstance(v, str)),
    "eps": ("a number", lambda v: hasattr(v, "__float__") and not isinstance(v, str)),
    "groups": ("an integer", lambda v: hasattr(v, "__index__")),
    "device": ("a ferrum_gpu.cuda.Device", lambda v: True),      # looked at by the call
    "stream": ("a stream", lambda v: True),
    **{name: ("a truth value", lambda v: hasattr(v, "__bool__"))
       for name in ("return_final_state", "delta_softplus", "save_states", "gate_inside")},
}


def _check_types(name, args):
    """Names the argument of the public function ``name`` that has a type its
    binding cannot take (both have their arguments in the same order)."""
    for arg, v in zip(inspect.signature(globals()[name]).parameters, args):
        if arg in _OTHERS:
            what, good = _OTHERS[arg]
            if not good(v):
                raise ValueError(f"{arg} must be {what}, got {type(v).__name__}")
        elif v is not None and not isinstance(v, torch.Tensor) and not hasattr(v, "__dlpack_device__"):
            raise ValueError(f"{arg} must be a CUDA tensor, got {type(v).__name__}")


def _from_dlpack(x, stream):
    place = getattr(x, "__dlpack_device__", None)
    if isinstance(x, torch.Tensor) or place is None:
        return x
    kind, ordinal = place()
    if kind != 2:   # kDLCUDA
        raise ValueError("tensor arguments must be a CUDA tensor (got one on the host)")
    # The producer orders its work in front of the stream that is current.
    with torch.cuda.stream(_torch_stream(stream, ordinal)):
        return torch.from_dlpack(x)


def _torch_stream(stream, ordinal):
    if stream is None or isinstance(stream, torch.cuda.Stream):
        return stream
    handle = int(getattr(stream, "cuda_stream", stream))
    return (torch.cuda.ExternalStream(handle, device=ordinal) if handle
            else torch.cuda.default_stream(ordinal))


# ---------------------------------------------------------------- short convolution

class ConvGrads(NamedTuple):
    dx: torch.Tensor
    dweight: torch.Tensor
    dbias: Optional[torch.Tensor]
    dinitial_state: Optional[torch.Tensor]


def causal_conv1d(x, weight, bias=None, *, activation=None, initial_state=None, lengths=None,
                  return_final_state=False, out=None, device=None, stream=None):
    """y[b,t,d] = act(bias[d] + sum_j weight[d,j] x[b,t-K+1+j,d]).

    x: (batch, length, channels). weight: (channels, taps). initial_state:
    (batch, taps - 1, channels) of x's type, the values in front of x, oldest
    first (zeros without it). Returns y, or (y, final_state) with the state a
    continuation starts from.
    """
    return _call(
        _sequence.causal_conv1d, x, weight, bias, activation, initial_state, lengths,
        return_final_state, out, device, stream)


def causal_conv1d_backward(dy, x, weight, bias=None, *, activation=None, initial_state=None,
                           lengths=None, dfinal_state=None, device=None, stream=None) -> ConvGrads:
    """Gradients of ``causal_conv1d`` for its output's gradient ``dy`` (and
    that of its final state). ``dbias`` and ``dinitial_state`` are None where
    the forward call had no bias or initial state."""
    return ConvGrads(*_call(
        _sequence.causal_conv1d_backward, dy, x, weight, bias, activation, initial_state,
        lengths, dfinal_state, device, stream))


def causal_conv1d_step(x, state, weight, bias=None, *, activation=None, next_state=None,
                       out=None, device=None, stream=None):
    """One step of every sequence. x: (batch, channels); state: (batch,
    taps - 1, channels), updated in place unless ``next_state`` takes the
    state after the step. Returns y (batch, channels)."""
    return _call(
        _sequence.causal_conv1d_step, x, state, weight, bias, activation, next_state, out,
        device, stream)


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
    return ScanResult(*_call(
        _sequence.selective_scan, u, delta, A, B, C, D, z, delta_bias, delta_softplus,
        initial_state, lengths, save_states, out, device, stream))


def selective_scan_backward(dout, u, delta, A, B, C, states, *, D=None, z=None, delta_bias=None,
                            delta_softplus=False, lengths=None, dfinal_state=None, device=None,
                            stream=None) -> ScanGrads:
    """Gradients of ``selective_scan`` for its output's gradient ``dout`` (and
    that of its final state). ``states`` comes from the forward call with
    ``save_states``. ``dD``, ``dz`` and ``ddelta_bias`` are None where the
    forward call lacked the argument."""
    return ScanGrads(*_call(
        _sequence.selective_scan_backward, dout, u, delta, A, B, C, states, D, z, delta_bias,
        delta_softplus, lengths, dfinal_state, device, stream))


def selective_scan_step(u, delta, A, B, C, state, *, D=None, z=None, delta_bias=None,
                        delta_softplus=False, next_state=None, out=None, device=None, stream=None):
    """One step of every sequence. u, delta, z: (batch, channels); B, C:
    (batch, states) or (batch, groups, states); state: (batch, channels,
    states) float32, updated in place unless ``next_state`` takes the state
    after the step. Returns out (batch, channels)."""
    return _call(
        _sequence.selective_scan_step, u, delta, A, B, C, state, D, z, delta_bias,
        delta_softplus, next_state, out, device, stream)


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


def norm_before(x, weight, bias=None, *, residual=None, scale=None, kind="rms", eps=1e-6,
                device=None, stream=None):
    """r = residual + scale * x;  y = N(r) * weight + bias.  Returns (y, r).

    x: (..., channels); residual: same shape, float32 or x's type, which r
    takes over (x's type without a residual); scale: (channels). N is
    v / sqrt(mean(v^2) + eps) ("rms") or (v - mean) / sqrt(var + eps)
    ("layer"). y has x's type.
    """
    return _call(_sequence.norm_before, x, weight, bias, residual, scale, kind, eps, device, stream)


def norm_before_backward(dy, r, weight, bias=None, *, dr=None, x=None, scale=None, kind="rms",
                         eps=1e-6, device=None, stream=None) -> NormBeforeGrads:
    """Gradients of ``norm_before`` for those of y (``dy``) and of r (``dr``,
    of r's type). ``r`` is the forward's; ``x`` is needed with ``scale``, for
    ``dscale``. ``dresidual`` has r's type, ``dx`` that of dy."""
    return NormBeforeGrads(*_call(
        _sequence.norm_before_backward, dy, r, weight, bias, dr, x, scale, kind, eps, device,
        stream))


def norm_after(x, weight, bias=None, *, gate=None, gate_inside=True, residual=None, scale=None,
               groups=1, kind="rms", eps=1e-6, out=None, device=None, stream=None):
    """residual + scale * p, with

        gate_inside:  p = N(x * silu(gate)) * weight + bias
        otherwise:    p = (N(x) * weight + bias) * silu(gate)

    x, gate: (..., channels) of one type; residual: float32 or x's type. N
    (see ``norm_before``) runs over each of ``groups`` equal parts of a row.
    """
    return _call(
        _sequence.norm_after, x, weight, bias, gate, gate_inside, residual, scale, groups, kind,
        eps, out, device, stream)


def norm_after_backward(dout, x, weight, bias=None, *, gate=None, gate_inside=True, scale=None,
                        groups=1, kind="rms", eps=1e-6, device=None, stream=None) -> NormAfterGrads:
    """Gradients of ``norm_after`` for its output's gradient ``dout``, which
    is also the gradient of the residual."""
    return NormAfterGrads(*_call(
        _sequence.norm_after_backward, dout, x, weight, bias, gate, gate_inside, scale, groups,
        kind, eps, device, stream))


# ---------------------------------------------------------------- long convolution

class LongGrads(NamedTuple):
    dx: torch.Tensor
    dkernel: torch.Tensor
    dskip: Optional[torch.Tensor]


def long_conv(x, kernel, skip=None, *, out=None, device=None, stream=None):
    """y[b,d,t] = sum_{s<=t} kernel[d,s] x[b,d,t-s] + skip[d] x[b,d,t].

    x: (batch, channels, length), any strides (contiguous length is fastest);
    kernel: (channels, taps), taps up to length; skip: (channels). Long rows go
    through the FFT, so an infinity or NaN reaches its whole row.
    """
    return _call(_sequence.long_conv, x, kernel, skip, out, device, stream)


def long_conv_backward(dy, x, kernel, skip=None, *, device=None, stream=None) -> LongGrads:
    """Gradients of ``long_conv``; ``dskip`` is None without ``skip``."""
    return LongGrads(*_call(_sequence.long_conv_backward, dy, x, kernel, skip, device, stream))


def long_conv_step(x, history, positions, kernel, skip=None, *, out=None, device=None, stream=None):
    """One token of every sequence. x: (batch, channels); history: (batch,
    channels, capacity) of x's type, contiguous along the last axis, holding
    the tokens before; positions: (batch) int32, where x goes. Stores x and
    returns y (batch, channels). A position outside the history stores nothing
    and its y is zero."""
    return _call(_sequence.long_conv_step, x, history, positions, kernel, skip, out, device, stream)


__all__ = ["causal_conv1d", "causal_conv1d_backward", "causal_conv1d_step", "selective_scan",
           "selective_scan_backward", "selective_scan_step", "norm_before", "norm_before_backward",
           "norm_after", "norm_after_backward", "long_conv", "long_conv_backward",
           "long_conv_step", "ConvGrads", "ScanResult", "ScanGrads", "NormBeforeGrads",
           "NormAfterGrads", "LongGrads"]
