"""Workloads of the sequence operators: the causal filters and norms of a
sequence-mixing block, next to the FFT.

Five operators, each in the directions a user calls it:

``conv``   short causal depthwise convolution with bias and SiLU
``scan``   selective state space scan (input-dependent linear recurrence)
``before`` residual update and norm in front of a block
``after``  gated norm behind a block with residual scale
``long``   causal convolution with a filter as long as the sequence

``mode`` is "forward", "train" (forward and gradients) or "step" (one token of
every sequence of a batch, on kept state). ``run`` computes them in plain torch
operations in 32 bits, or, where ``own`` is true, through ``ferrum_gpu.sequence``.
"""

import math
import sys

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # One token of one conversation: the smallest call, all latency.
        dict(name="scan_step_1", op="scan", mode="step", dtype="bf16", batch=1, length=1,
             channels=2048, states=16, groups=1, ragged=False),
        # One token of a full serving batch.
        dict(name="conv_step_256", op="conv", mode="step", dtype="bf16", batch=256, length=1,
             channels=4096, taps=4, silu=True, ragged=False),
        # The same serving batch's state update.
        dict(name="scan_step_256", op="scan", mode="step", dtype="f16", batch=256, length=1,
             channels=4096, states=16, groups=1, ragged=False),
        # One long prompt: few rows, a long axis.
        dict(name="scan_prompt", op="scan", mode="forward", dtype="bf16", batch=1, length=8191,
             channels=2048, states=16, groups=1, ragged=False),
        # A batch of prompts of different lengths, odd sizes, full precision.
        dict(name="scan_ragged", op="scan", mode="forward", dtype="f32", batch=13, length=777,
             channels=1000, states=16, groups=2, ragged=True),
        # The training step's scan: the largest work.
        dict(name="scan_train", op="scan", mode="train", dtype="bf16", batch=8, length=2048,
             channels=2048, states=16, groups=1, ragged=False),
        # The training step's short convolution.
        dict(name="conv_train", op="conv", mode="train", dtype="bf16", batch=8, length=2048,
             channels=4096, taps=4, silu=True, ragged=False),
        # Norm in front of a block for a small decode batch.
        dict(name="before_decode", op="before", mode="forward", dtype="bf16", rows=32,
             channels=4096, kind="rms"),
        # Norm in front of a block in training, 32-bit residual stream.
        dict(name="before_train", op="before", mode="train", dtype="bf16", rows=16384,
             channels=2048, kind="rms"),
        # Gated norm in groups behind a block in training, an odd number of rows.
        dict(name="after_train", op="after", mode="train", dtype="bf16", rows=8191,
             channels=4096, groups=8, kind="rms", inside=True),
        # Long filters over a batch of sequences of a single-pass FFT length.
        dict(name="long_forward", op="long", mode="forward", dtype="bf16", batch=8, length=4096,
             channels=1024),
        # The same in training, a length that is no power of two.
        dict(name="long_train", op="long", mode="train", dtype="f32", batch=2, length=6000,
             channels=384),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["conv", "scan", "scan", "before", "after", "long"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "conv":
        mode = rng.choice(["forward", "train", "step"])
        channels = _log_int(rng, 64, 5000)
        batch = _log_int(rng, 1, 256 if mode == "step" else 16)
        limit = 60_000_000 // (channels * batch)
        length = 1 if mode == "step" else _log_int(rng, 1, max(1, min(16384, limit)))
        return dict(op=op, mode=mode, dtype=dtype, batch=batch, length=length, channels=channels,
                    taps=rng.choice([2, 3, 4, 4]), silu=rng.random() < 0.8,
                    ragged=mode != "step" and rng.random() < 0.3)
    if op == "scan":
        mode = rng.choice(["forward", "train", "step"])
        states = rng.choice([8, 16, 16, 16, 13, 32])
        groups = rng.choice([1, 1, 2])
        channels = _log_int(rng, 64, 4200)
        channels -= channels % groups
        batch = _log_int(rng, 1, 256 if mode == "step" else 16)
        limit = (500_000_000 if mode != "train" else 250_000_000) // (channels * batch * states)
        length = 1 if mode == "step" else _log_int(rng, 1, max(1, min(8192 if mode == "forward" else 2048, limit)))
        return dict(op=op, mode=mode, dtype=dtype, batch=batch, length=length, channels=channels,
                    states=states, groups=groups, ragged=mode != "step" and rng.random() < 0.3)
    if op == "before":
        mode = rng.choice(["forward", "train"])
        channels = _log_int(rng, 64, 8192)
        rows = _log_int(rng, 1, max(1, min(32768, 30_000_000 // channels)))
        return dict(op=op, mode=mode, dtype=dtype, rows=rows, channels=channels,
                    kind=rng.choice(["rms", "rms", "layer"]))
    if op == "after":
        mode = rng.choice(["forward", "train"])
        groups = rng.choice([1, 1, 4, 8])
        channels = groups * _log_int(rng, 32, 8192 // groups)
        rows = _log_int(rng, 1, max(1, min(32768, 30_000_000 // channels)))
        return dict(op=op, mode=mode, dtype=dtype, rows=rows, channels=channels, groups=groups,
                    kind=rng.choice(["rms", "rms", "layer"]), inside=rng.random() < 0.5)
    mode = rng.choice(["forward", "train", "step"])
    if mode == "step":
        batch, channels = _log_int(rng, 1, 64), _log_int(rng, 64, 1024)
        length = _log_int(rng, 1, max(1, min(8192, 60_000_000 // (batch * channels))))
    else:
        batch = _log_int(rng, 1, 8)
        length = _log_int(rng, 2, 16384)
        cap = 8_000_000_000 if mode == "forward" else 4_000_000_000
        channels = _log_int(rng, 16, max(16, min(1024, cap // (length * length),
                                                 30_000_000 // (batch * length))))
    return dict(op=op, mode=mode, dtype=dtype, batch=batch, length=length, channels=channels)


# ---------------------------------------------------------------- inputs

class _Rand:
    """Seeded random tensors on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def normal(self, shape, dtype=torch.float32, std=1.0):
        return (torch.randn(shape, generator=self.g, device="cuda") * std).to(dtype)

    def uniform(self, shape, lo, hi):
        return torch.rand(shape, generator=self.g, device="cuda") * (hi - lo) + lo


def _lengths(case, r):
    if not case.get("ragged"):
        return None
    b, n = case["batch"], case["length"]
    out = torch.floor(r.uniform((b,), 0, n + 1)).to(torch.int32).clamp_(0, n)
    out[0] = n                       # one sequence fills the batch's length,
    if b > 2:
        out[b // 2] = 0              # one is empty
    return out


def prepare(case, seed):
    r = _Rand(seed)
    dt = _DTYPES[case["dtype"]]
    op, mode = case["op"], case["mode"]
    s = {"case": case}
    if op in ("conv", "scan"):
        b, n, d = case["batch"], case["length"], case["channels"]
        lead = (b, d) if mode == "step" else (b, n, d)
        s["lengths"] = _lengths(case, r)
        if op == "conv":
            k = case["taps"]
            s["x"] = r.normal(lead, dt)
            s["weight"] = r.normal((d, k), std=1.0 / math.sqrt(k))
            s["bias"] = r.normal((d,), std=0.1)
            # a prompt that continues an earlier one starts from its last taps
            s["state"] = r.normal((b, k - 1, d), dt)
            if mode == "train":
                s["dy"] = r.normal(lead, dt)
            if mode == "step":
                s["next_state"] = torch.empty_like(s["state"])
        else:
            st, g = case["states"], case["groups"]
            s["u"] = r.normal(lead, dt)
            s["z"] = r.normal(lead, dt)
            s["delta"] = r.normal(lead, dt, 0.5)
            step = torch.exp(r.uniform((d,), math.log(1e-3), math.log(1e-1)))
            s["delta_bias"] = step + torch.log(-torch.expm1(-step))
            decay = torch.arange(1, st + 1, device="cuda", dtype=torch.float32).expand(d, st)
            s["A"] = (-decay * torch.exp(r.normal((d, st), std=0.1))).contiguous()
            s["B"] = r.normal(lead[:-1] + (g, st), dt)
            s["C"] = r.normal(lead[:-1] + (g, st), dt)
            s["D"] = r.normal((d,), std=0.5)
            s["state"] = r.normal((b, d, st), std=0.3)
            if mode == "train":
                s["dout"] = r.normal(lead, dt)
            if mode == "step":
                s["next_state"] = torch.empty_like(s["state"])
    elif op == "before":
        m, d = case["rows"], case["channels"]
        s["x"] = r.normal((m, d), dt)
        s["residual"] = r.normal((m, d), std=2.0)
        s["scale"] = r.normal((d,), std=0.1) + 0.5
        s["weight"] = r.normal((d,), std=0.1) + 1.0
        s["bias"] = r.normal((d,), std=0.1) if case["kind"] == "layer" else None
        if mode == "train":
            s["dy"] = r.normal((m, d), dt)
            s["dr"] = r.normal((m, d))
    elif op == "after":
        m, d = case["rows"], case["channels"]
        s["x"] = r.normal((m, d), dt)
        s["gate"] = r.normal((m, d), dt)
        s["residual"] = r.normal((m, d), dt)
        s["scale"] = r.normal((d,), std=0.1) + 0.5
        s["weight"] = r.normal((d,), std=0.1) + 1.0
        s["bias"] = r.normal((d,), std=0.1) if case["kind"] == "layer" else None
        if mode == "train":
            s["dout"] = r.normal((m, d), dt)
    else:
        b, n, d = case["batch"], case["length"], case["channels"]
        fade = torch.exp(-torch.arange(n, device="cuda") * (4.0 / n))
        s["kernel"] = r.normal((d, n), std=1.0 / math.sqrt(n)) * fade
        s["skip"] = r.normal((d,), std=0.5)
        if mode == "step":
            # `length` tokens are kept per sequence, the last one arrives now
            s["x"] = r.normal((b, d), dt)
            s["history"] = r.normal((b, d, n), dt)
            s["positions"] = torch.floor(r.uniform((b,), 0, n)).to(torch.int32).clamp_(0, n - 1)
            s["positions"][0] = n - 1
        else:
            s["x"] = r.normal((b, d, n), dt)
            if mode == "train":
                s["dy"] = r.normal((b, d, n), dt)
    if own:
        _sequence()
    return s


# ---------------------------------------------------------------- one pass

def run(state):
    case = state["case"]
    which = _OWN if own else _PLAIN
    return which[(case["op"], case["mode"])](state, case)


def _sequence():
    if "ferrum-gpu_b200" not in sys.path:
        sys.path.insert(0, "ferrum-gpu_b200")
    from ferrum_gpu import sequence

    return sequence


# The framework's calls.

def _own_conv_forward(s, c):
    y, fin = _sequence().causal_conv1d(s["x"], s["weight"], s["bias"],
                                       activation="silu" if c["silu"] else None,
                                       initial_state=s["state"], lengths=s["lengths"],
                                       return_final_state=True)
    return {"y": y, "state": fin}


def _own_conv_train(s, c):
    seq = _sequence()
    act = "silu" if c["silu"] else None
    y, fin = seq.causal_conv1d(s["x"], s["weight"], s["bias"], activation=act,
                               initial_state=s["state"], lengths=s["lengths"],
                               return_final_state=True)
    g = seq.causal_conv1d_backward(s["dy"], s["x"], s["weight"], s["bias"], activation=act,
                                   initial_state=s["state"], lengths=s["lengths"])
    return {"y": y, "state": fin, "dx": g.dx, "dweight": g.dweight, "dbias": g.dbias,
            "dstate": g.dinitial_state}


def _own_conv_step(s, c):
    y = _sequence().causal_conv1d_step(s["x"], s["state"], s["weight"], s["bias"],
                                       activation="silu" if c["silu"] else None,
                                       next_state=s["next_state"])
    return {"y": y, "state": s["next_state"]}


def _own_scan_forward(s, c):
    r = _sequence().selective_scan(s["u"], s["delta"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"],
                                   delta_bias=s["delta_bias"], delta_softplus=True,
                                   initial_state=s["state"], lengths=s["lengths"])
    return {"out": r.out, "state": r.final_state}


def _own_scan_train(s, c):
    seq = _sequence()
    r = seq.selective_scan(s["u"], s["delta"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"],
                           delta_bias=s["delta_bias"], delta_softplus=True,
                           initial_state=s["state"], lengths=s["lengths"], save_states=True)
    g = seq.selective_scan_backward(s["dout"], s["u"], s["delta"], s["A"], s["B"], s["C"],
                                    r.states, D=s["D"], z=s["z"], delta_bias=s["delta_bias"],
                                    delta_softplus=True, lengths=s["lengths"])
    return {"out": r.out, "state": r.final_state, "du": g.du, "ddelta": g.ddelta, "dA": g.dA,
            "dB": g.dB, "dC": g.dC, "dD": g.dD, "dz": g.dz, "ddelta_bias": g.ddelta_bias,
            "dstate": g.dinitial_state}


def _own_scan_step(s, c):
    y = _sequence().selective_scan_step(s["u"], s["delta"], s["A"], s["B"], s["C"], s["state"],
                                        D=s["D"], z=s["z"], delta_bias=s["delta_bias"],
                                        delta_softplus=True, next_state=s["next_state"])
    return {"out": y, "state": s["next_state"]}


def _own_before_forward(s, c):
    y, r = _sequence().norm_before(s["x"], s["weight"], s["bias"], residual=s["residual"],
                                   scale=s["scale"], kind=c["kind"], eps=1e-6)
    return {"y": y, "r": r}


def _own_before_train(s, c):
    seq = _sequence()
    y, r = seq.norm_before(s["x"], s["weight"], s["bias"], residual=s["residual"],
                           scale=s["scale"], kind=c["kind"], eps=1e-6)
    g = seq.norm_before_backward(s["dy"], r, s["weight"], s["bias"], dr=s["dr"], x=s["x"],
                                 scale=s["scale"], kind=c["kind"], eps=1e-6)
    return {"y": y, "r": r, "dx": g.dx, "dresidual": g.dresidual, "dweight": g.dweight,
            "dbias": g.dbias, "dscale": g.dscale}


def _own_after_forward(s, c):
    return {"out": _sequence().norm_after(
        s["x"], s["weight"], s["bias"], gate=s["gate"], gate_inside=c["inside"],
        residual=s["residual"], scale=s["scale"], groups=c["groups"], kind=c["kind"], eps=1e-6)}


def _own_after_train(s, c):
    seq = _sequence()
    out = seq.norm_after(s["x"], s["weight"], s["bias"], gate=s["gate"], gate_inside=c["inside"],
                         residual=s["residual"], scale=s["scale"], groups=c["groups"],
                         kind=c["kind"], eps=1e-6)
    g = seq.norm_after_backward(s["dout"], s["x"], s["weight"], s["bias"], gate=s["gate"],
                                gate_inside=c["inside"], scale=s["scale"], groups=c["groups"],
                                kind=c["kind"], eps=1e-6)
    return {"out": out, "dx": g.dx, "dgate": g.dgate, "dweight": g.dweight, "dbias": g.dbias,
            "dscale": g.dscale}


def _own_long_forward(s, c):
    return {"y": _sequence().long_conv(s["x"], s["kernel"], s["skip"])}


def _own_long_train(s, c):
    seq = _sequence()
    y = seq.long_conv(s["x"], s["kernel"], s["skip"])
    g = seq.long_conv_backward(s["dy"], s["x"], s["kernel"], s["skip"])
    return {"y": y, "dx": g.dx, "dkernel": g.dkernel, "dskip": g.dskip}


def _own_long_step(s, c):
    y = _sequence().long_conv_step(s["x"], s["history"], s["positions"], s["kernel"], s["skip"])
    return {"y": y, "history": s["history"]}


# The plain forms.

def _silu(x):
    return x / (1.0 + torch.exp(-x))


def _dsilu(x):
    g = 1.0 / (1.0 + torch.exp(-x))
    return g * (1.0 + x * (1.0 - g))


def _softplus(x):
    return torch.clamp(x, min=0.0) + torch.log1p(torch.exp(-torch.abs(x)))


def _valid(s, n):
    """(batch, length, 1) truth values: the steps inside each sequence."""
    t = torch.arange(n, device="cuda")
    if s["lengths"] is None:
        return torch.ones((1, n, 1), dtype=torch.bool, device="cuda")
    return (t[None, :] < s["lengths"][:, None])[:, :, None]


def _zero(x, keep):
    return torch.where(keep, x, torch.zeros((), device=x.device, dtype=x.dtype))


def _plain_conv(s, c):
    x, w = s["x"].float(), s["weight"]
    b, n, d = x.shape
    k = c["taps"]
    keep = _valid(s, n)
    x = _zero(x, keep)
    full = torch.cat([s["state"].float(), x], dim=1)
    pre = s["bias"] + sum(w[:, j] * full[:, j:j + n] for j in range(k))
    y = _zero(_silu(pre) if c["silu"] else pre, keep)
    ends = (s["lengths"].long() if s["lengths"] is not None
            else torch.full((b,), n, device="cuda"))
    idx = ends[:, None] + torch.arange(k - 1, device="cuda")[None, :]
    fin = full[torch.arange(b, device="cuda")[:, None], idx]
    return x, keep, full, pre, y, fin


def _plain_conv_forward(s, c):
    dt = s["x"].dtype
    _, _, _, _, y, fin = _plain_conv(s, c)
    return {"y": y.to(dt), "state": fin.to(dt)}


def _plain_conv_train(s, c):
    dt, w, k = s["x"].dtype, s["weight"], c["taps"]
    x, keep, full, pre, y, fin = _plain_conv(s, c)
    n = x.shape[1]
    g = s["dy"].float() * (_dsilu(pre) if c["silu"] else 1.0)
    g = _zero(g, keep)
    dfull = torch.zeros_like(full)
    for j in range(k):
        dfull[:, j:j + n] += w[:, j] * g
    dw = torch.stack([(g * full[:, j:j + n]).sum((0, 1)) for j in range(k)], dim=1)
    return {"y": y.to(dt), "state": fin.to(dt), "dx": _zero(dfull[:, k - 1:], keep).to(dt),
            "dweight": dw, "dbias": g.sum((0, 1)), "dstate": dfull[:, :k - 1].to(dt)}


def _plain_conv_step(s, c):
    dt = s["x"].dtype
    full = torch.cat([s["state"].float(), s["x"].float()[:, None]], dim=1)
    pre = s["bias"] + (full * s["weight"].t()).sum(1)
    return {"y": (_silu(pre) if c["silu"] else pre).to(dt), "state": full[:, 1:].to(dt)}


def _spread(x, d):
    """(..., groups, states) of the channels' groups to (..., channels, states)."""
    return x.repeat_interleave(d // x.shape[-2], dim=-2)


def _plain_scan(s, c, keep_all):
    u, z = s["u"].float(), s["z"].float()
    n, d = u.shape[1], u.shape[2]
    keep = _valid(s, n)
    dt = _softplus(s["delta"].float() + s["delta_bias"])
    h = s["state"]
    ys, hs = [], [h]
    for t in range(n):
        a = torch.exp(dt[:, t, :, None] * s["A"])
        bt = _spread(s["B"][:, t].float(), d)
        ct = _spread(s["C"][:, t].float(), d)
        nxt = a * h + (dt[:, t] * u[:, t])[:, :, None] * bt
        h = nxt if s["lengths"] is None else torch.where(keep[:, t, :, None], nxt, h)
        ys.append((h * ct).sum(-1))
        if keep_all:
            hs.append(h)
    y = torch.stack(ys, dim=1) + s["D"] * u
    return u, z, dt, keep, y, h, hs


def _plain_scan_forward(s, c):
    _, z, _, keep, y, h, _ = _plain_scan(s, c, False)
    return {"out": _zero(y * _silu(z), keep).to(s["u"].dtype), "state": h}


def _plain_scan_train(s, c):
    dtype = s["u"].dtype
    u, z, dt, keep, y, fin, hs = _plain_scan(s, c, True)
    b, n, d = u.shape
    g, st = c["groups"], c["states"]
    dout = _zero(s["dout"].float(), keep)
    dz = dout * y * _dsilu(z)
    dy = dout * _silu(z)
    du, ddt = dy * s["D"], torch.zeros_like(u)
    dA = torch.zeros_like(s["A"])
    dB, dC = (torch.zeros((b, n, g, st), device="cuda") for _ in range(2))
    gh = torch.zeros_like(fin)
    for t in range(n - 1, -1, -1):
        live = keep[:, t, :, None]
        a = torch.exp(dt[:, t, :, None] * s["A"])
        bt = _spread(s["B"][:, t].float(), d)
        ct = _spread(s["C"][:, t].float(), d)
        cur = gh + ct * dy[:, t, :, None]
        if s["lengths"] is not None:
            cur = torch.where(live, cur, torch.zeros((), device="cuda"))
        dC[:, t] = (dy[:, t, :, None] * hs[t + 1]).reshape(b, g, d // g, st).sum(2)
        dB[:, t] = (cur * (dt[:, t] * u[:, t])[:, :, None]).reshape(b, g, d // g, st).sum(2)
        gb = (cur * bt).sum(-1)
        du[:, t] += gb * dt[:, t]
        gah = cur * a * hs[t]
        ddt[:, t] = (gah * s["A"]).sum(-1) + gb * u[:, t]
        dA += (gah * dt[:, t, :, None]).sum(0)
        gh = cur * a if s["lengths"] is None else torch.where(live, cur * a, gh)
    slope = 1.0 / (1.0 + torch.exp(-(s["delta"].float() + s["delta_bias"])))
    ddelta = _zero(ddt * slope, keep)
    return {"out": _zero(y * _silu(z), keep).to(dtype), "state": fin,
            "du": _zero(du, keep).to(dtype), "ddelta": ddelta.to(dtype), "dA": dA,
            "dB": dB.to(dtype), "dC": dC.to(dtype), "dD": (dy * u).sum((0, 1)),
            "dz": dz.to(dtype), "ddelta_bias": ddelta.sum((0, 1)), "dstate": gh}


def _plain_scan_step(s, c):
    u, z = s["u"].float(), s["z"].float()
    d = u.shape[1]
    dt = _softplus(s["delta"].float() + s["delta_bias"])
    h = (torch.exp(dt[:, :, None] * s["A"]) * s["state"]
         + (dt * u)[:, :, None] * _spread(s["B"].float(), d))
    y = (h * _spread(s["C"].float(), d)).sum(-1) + s["D"] * u
    return {"out": (y * _silu(z)).to(s["u"].dtype), "state": h}


def _normed(v, kind):
    """The normalised rows and 1 / deviation."""
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    inv = 1.0 / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-6)
    return v * inv, inv


def _norm_grad(dn, n, inv, kind):
    """Gradient of the norm's input from that of its output."""
    out = dn - n * (dn * n).mean(-1, keepdim=True)
    if kind == "layer":
        out = out - dn.mean(-1, keepdim=True)
    return out * inv


def _plain_before(s, c):
    r = s["residual"] + s["scale"] * s["x"].float()
    n, inv = _normed(r, c["kind"])
    y = n * s["weight"]
    return r, n, inv, (y if s["bias"] is None else y + s["bias"])


def _plain_before_forward(s, c):
    r, _, _, y = _plain_before(s, c)
    return {"y": y.to(s["x"].dtype), "r": r}


def _plain_before_train(s, c):
    r, n, inv, y = _plain_before(s, c)
    dy = s["dy"].float()
    dr = _norm_grad(dy * s["weight"], n, inv, c["kind"]) + s["dr"]
    return {"y": y.to(s["x"].dtype), "r": r, "dx": (dr * s["scale"]).to(s["x"].dtype),
            "dresidual": dr, "dweight": (dy * n).sum(0),
            "dbias": None if s["bias"] is None else dy.sum(0),
            "dscale": (dr * s["x"].float()).sum(0)}


def _plain_after(s, c):
    m, d = s["x"].shape
    x, gate = s["x"].float(), s["gate"].float()
    v = x * _silu(gate) if c["inside"] else x
    n, inv = _normed(v.reshape(m, c["groups"], -1), c["kind"])
    w = n.reshape(m, d) * s["weight"]
    if s["bias"] is not None:
        w = w + s["bias"]
    p = w if c["inside"] else w * _silu(gate)
    return x, gate, n, inv, w, p


def _plain_after_forward(s, c):
    p = _plain_after(s, c)[-1]
    return {"out": (s["residual"].float() + s["scale"] * p).to(s["x"].dtype)}


def _plain_after_train(s, c):
    m, d = s["x"].shape
    dt = s["x"].dtype
    x, gate, n, inv, w, p = _plain_after(s, c)
    dout = s["dout"].float()
    dw = dout * s["scale"]
    dgate = None
    if not c["inside"]:
        dgate = dw * w * _dsilu(gate)
        dw = dw * _silu(gate)
    dn = (dw * s["weight"]).reshape(m, c["groups"], -1)
    dv = _norm_grad(dn, n, inv, c["kind"]).reshape(m, d)
    if c["inside"]:
        dgate = dv * x * _dsilu(gate)
        dv = dv * _silu(gate)
    return {"out": (s["residual"].float() + s["scale"] * p).to(dt), "dx": dv.to(dt),
            "dgate": dgate.to(dt), "dweight": (dw * n.reshape(m, d)).sum(0),
            "dbias": None if s["bias"] is None else dw.sum(0), "dscale": (dout * p).sum(0)}


def _lagged(v, n):
    """(rows, n, n) with [t, s] = v[t - s] for s <= t, else 0."""
    t = torch.arange(n, device="cuda")
    lag = t[:, None] - t[None, :]
    return torch.where(lag >= 0, v[:, lag.clamp(min=0)], torch.zeros((), device="cuda"))


def _blocks(total, n):
    step = max(1, (1 << 28) // (n * n))
    return [slice(i, min(total, i + step)) for i in range(0, total, step)]


def _plain_long_forward(s, c):
    x = s["x"].float()
    y = torch.empty_like(x)
    for q in _blocks(x.shape[1], x.shape[2]):
        lag = _lagged(s["kernel"][q], x.shape[2])
        y[:, q] = (lag @ x[:, q].permute(1, 2, 0)).permute(2, 0, 1)
    return {"y": (y + s["skip"][:, None] * x).to(s["x"].dtype)}


def _plain_long_train(s, c):
    x, dy = s["x"].float(), s["dy"].float()
    b, d, n = x.shape
    dx, dk = torch.empty_like(x), torch.zeros_like(s["kernel"])
    for q in _blocks(d, n):
        lag = _lagged(s["kernel"][q], n)
        dx[:, q] = (lag.transpose(1, 2) @ dy[:, q].permute(1, 2, 0)).permute(2, 0, 1)
        for i in range(b):
            dk[q] += (_lagged(x[i, q], n).transpose(1, 2) @ dy[i, q, :, None])[:, :, 0]
    return {"y": _plain_long_forward(s, c)["y"],
            "dx": (dx + s["skip"][:, None] * dy).to(s["x"].dtype), "dkernel": dk,
            "dskip": (x * dy).sum((0, 2))}


def _plain_long_step(s, c):
    x, hist, pos = s["x"].float(), s["history"], s["positions"].long()
    b, d, n = hist.shape
    t = torch.arange(n, device="cuda")
    lag = pos[:, None] - t[None, :]
    here = (lag == 0)[:, None, :]
    hist = torch.where(here, s["x"][:, :, None], hist)
    taps = torch.where((lag >= 0)[None], s["kernel"][:, lag.clamp(min=0)],
                       torch.zeros((), device="cuda")).transpose(0, 1)
    y = (taps * torch.where((lag >= 0)[:, None], hist.float(),
                            torch.zeros((), device="cuda"))).sum(-1)
    return {"y": (y + s["skip"] * x).to(s["x"].dtype), "history": hist}


_PLAIN = {("conv", "forward"): _plain_conv_forward, ("conv", "train"): _plain_conv_train,
          ("conv", "step"): _plain_conv_step, ("scan", "forward"): _plain_scan_forward,
          ("scan", "train"): _plain_scan_train, ("scan", "step"): _plain_scan_step,
          ("before", "forward"): _plain_before_forward, ("before", "train"): _plain_before_train,
          ("after", "forward"): _plain_after_forward, ("after", "train"): _plain_after_train,
          ("long", "forward"): _plain_long_forward, ("long", "train"): _plain_long_train,
          ("long", "step"): _plain_long_step}
_OWN = {("conv", "forward"): _own_conv_forward, ("conv", "train"): _own_conv_train,
        ("conv", "step"): _own_conv_step, ("scan", "forward"): _own_scan_forward,
        ("scan", "train"): _own_scan_train, ("scan", "step"): _own_scan_step,
        ("before", "forward"): _own_before_forward, ("before", "train"): _own_before_train,
        ("after", "forward"): _own_after_forward, ("after", "train"): _own_after_train,
        ("long", "forward"): _own_long_forward, ("long", "train"): _own_long_train,
        ("long", "step"): _own_long_step}


# ---------------------------------------------------------------- work

def work(case):
    """Bytes each pass has to move (inputs once, outputs once) and its
    arithmetic; an exponential, a product and a sum count one each."""
    e = _BYTES[case["dtype"]]
    op, mode = case["op"], case["mode"]
    train = mode == "train"
    if op == "conv":
        b, d, k = case["batch"], case["channels"], case["taps"]
        cells = b * case["length"] * d
        params = 4 * d * (k + 1)
        states = 2 * b * (k - 1) * d * e
        if train:       # x and dy in, y and dx out
            return {"bytes": 4 * cells * e + 2 * params + states * 3 // 2,
                    "flops": cells * (6 * k + 16)}
        return {"bytes": 2 * cells * e + params + states, "flops": cells * (2 * k + 5)}
    if op == "scan":
        b, d, n, g = case["batch"], case["channels"], case["states"], case["groups"]
        cells = b * case["length"] * d
        shared = 2 * b * case["length"] * g * n * e
        params = 4 * d * (n + 2)
        states = 2 * 4 * b * d * n
        if train:       # u, delta, z, dout in; out, du, ddelta, dz out
            return {"bytes": 8 * cells * e + 2 * shared + 2 * params + states * 3 // 2,
                    "flops": cells * (22 * n + 40)}
        return {"bytes": 4 * cells * e + shared + params + states, "flops": cells * (6 * n + 14)}
    if op == "before":
        m, d = case["rows"], case["channels"]
        params = 4 * d * (3 if case["kind"] == "layer" else 2)
        if train:       # x, residual, dy, dr in; y, r, dx, dresidual out
            return {"bytes": m * d * (4 * e + 16) + 2 * params, "flops": m * d * 22}
        return {"bytes": m * d * (2 * e + 8) + params, "flops": m * d * 7}
    if op == "after":
        m, d = case["rows"], case["channels"]
        params = 4 * d * (3 if case["kind"] == "layer" else 2)
        if train:       # x, gate, residual, dout in; out, dx, dgate out
            return {"bytes": m * d * 7 * e + 2 * params, "flops": m * d * 40}
        return {"bytes": m * d * 4 * e + params, "flops": m * d * 14}
    b, n, d = case["batch"], case["length"], case["channels"]
    if mode == "step":
        # on average half of the kept tokens lie before the positions
        return {"bytes": b * d * (n * e // 2 + 3 * e) + 4 * d * (n + 1), "flops": b * d * n}
    m = max(2, 1 << (n - 1).bit_length())
    fft = 5 * m * int(math.log2(m))
    if train:           # x, dy in; y, dx out; the transforms x, dy, y, dx per row, k, dk per channel
        return {"bytes": 4 * b * d * n * e + 8 * d * (n + 1),
                "flops": b * d * (4 * fft + 50 * m) + 2 * d * fft}
    return {"bytes": 2 * b * d * n * e + 4 * d * (n + 1),
            "flops": b * d * (2 * fft + 16 * m) + d * fft}


# ---------------------------------------------------------------- 64 bits

def exact(case, seed):
    """``run``'s outputs from the definitions in 64 bits; gradients come from
    differentiating the definition."""
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    return _EXACT[case["op"]](s, case)


def _leaf(x):
    return None if x is None else x.double().requires_grad_(True)


def _grads(loss, leaves):
    live = {k: v for k, v in leaves.items() if v is not None}
    got = torch.autograd.grad(loss, list(live.values()))
    return {**{k: None for k in leaves}, **dict(zip(live, (g.detach() for g in got)))}


def _exact_conv(s, c):
    k, step, train = c["taps"], c["mode"] == "step", c["mode"] == "train"
    x = s["x"][:, None] if step else s["x"]
    b, n, d = x.shape
    ends = (s["lengths"].long() if s["lengths"] is not None else
            torch.full((b,), n, device="cuda", dtype=torch.long))
    inside = (torch.arange(n, device="cuda") < ends[:, None])[..., None]
    v = {"x": _leaf(x), "weight": _leaf(s["weight"]), "bias": _leaf(s["bias"]),
         "state": _leaf(s["state"])}
    with torch.set_grad_enabled(train):
        line = torch.cat([v["state"], v["x"].masked_fill(~inside, 0.0)], 1)
        pre = torch.einsum("bndk,dk->bnd", line.unfold(1, k, 1), v["weight"]) + v["bias"]
        y = (pre * torch.sigmoid(pre) if c["silu"] else pre).masked_fill(~inside, 0.0)
    fin = torch.stack([line[i, e:e + k - 1] for i, e in enumerate(ends.tolist())]).detach()
    out = {"y": y.detach()[:, 0] if step else y.detach(), "state": fin}
    if train:
        dy = s["dy"].double().masked_fill(~inside, 0.0)
        g = _grads((y * dy).sum(), v)
        out.update(dx=g["x"], dweight=g["weight"], dbias=g["bias"], dstate=g["state"])
    return out


def _exact_scan_part(s, c, q, grp):
    """Channels `q`, all of group `grp`, by doubling: after round i each step
    holds the composition of the last 2^i steps' maps h -> a h + b."""
    step, train = c["mode"] == "step", c["mode"] == "train"
    cut = (lambda x: x[:, None]) if step else (lambda x: x)
    v = {"u": _leaf(cut(s["u"])[..., q]), "delta": _leaf(cut(s["delta"])[..., q]),
         "z": _leaf(cut(s["z"])[..., q]), "A": _leaf(s["A"][q]), "D": _leaf(s["D"][q]),
         "bias": _leaf(s["delta_bias"][q]), "state": _leaf(s["state"][:, q]),
         "B": _leaf(cut(s["B"])[..., grp, :]), "C": _leaf(cut(s["C"])[..., grp, :])}
    n = v["u"].shape[1]
    with torch.set_grad_enabled(train):
        dt = torch.nn.functional.softplus(v["delta"] + v["bias"], threshold=50.0)
        if s["lengths"] is not None:
            inside = (torch.arange(n, device="cuda") < s["lengths"][:, None])[..., None]
            dt = dt.masked_fill(~inside, 0.0)      # a = 1, b = 0: the state stands still
        b = (dt * v["u"])[..., None] * v["B"][:, :, None]
        log_a = dt[..., None] * v["A"]
        a = torch.exp(log_a)
        first = torch.zeros_like(b)
        first[:, 0] = 1.0
        b = b + first * (a[:, :1] * v["state"][:, None])
        reach = 1
        while reach < n:
            b = torch.cat([b[:, :reach], b[:, reach:] + a[:, reach:] * b[:, :-reach]], 1)
            a = torch.cat([a[:, :reach], a[:, reach:] * a[:, :-reach]], 1)
            reach *= 2
        y = torch.einsum("bldn,bln->bld", b, v["C"]) + v["D"] * v["u"]
        out = y * v["z"] * torch.sigmoid(v["z"])
        if s["lengths"] is not None:
            out = out.masked_fill(~inside, 0.0)
    got = {"out": out.detach(), "state": b[:, -1].detach().clone()}
    if train:
        g = _grads((out * s["dout"][..., q].double()).sum(), v)
        got.update(du=g["u"], ddelta=g["delta"], dA=g["A"], dB=g["B"], dC=g["C"], dD=g["D"],
                   dz=g["z"], ddelta_bias=g["bias"], dstate=g["state"])
    if step:
        got["out"] = got["out"][:, 0]
    return got


def _exact_scan(s, c):
    d, g = c["channels"], c["groups"]
    per = d // g
    width = max(1, min(per, (1 << 25) // max(1, c["batch"] * c["length"] * c["states"])))
    axis = {"out": -1, "state": 1, "du": -1, "ddelta": -1, "dA": 0, "dD": 0, "dz": -1,
            "ddelta_bias": 0, "dstate": 1}
    parts, shared = [], {"dB": [], "dC": []}
    for grp in range(g):
        sums = {}
        for lo in range(grp * per, (grp + 1) * per, width):
            p = _exact_scan_part(s, c, slice(lo, min(lo + width, (grp + 1) * per)), grp)
            for k in shared:
                if k in p:
                    sums[k] = sums[k] + p.pop(k) if k in sums else p.pop(k)
            parts.append(p)
        for k in sums:
            shared[k].append(sums[k])
    out = {k: torch.cat([p[k] for p in parts], axis[k]) for k in parts[0]}
    out.update({k: torch.stack(v, 2) for k, v in shared.items() if v})
    order = ["out", "state", "du", "ddelta", "dA", "dB", "dC", "dD", "dz", "ddelta_bias", "dstate"]
    return {k: out[k] for k in order if k in out}


def _exact_norm(v, kind):
    if kind == "layer":
        var, mean = torch.var_mean(v, dim=-1, correction=0, keepdim=True)
        return (v - mean) / torch.sqrt(var + 1e-6)
    return v * torch.rsqrt(v.pow(2).mean(-1, keepdim=True) + 1e-6)


def _exact_before(s, c):
    train = c["mode"] == "train"
    v = {k: _leaf(s[k]) for k in ("x", "residual", "weight", "bias", "scale")}
    with torch.set_grad_enabled(train):
        r = torch.addcmul(v["residual"], v["scale"].expand_as(v["x"]), v["x"])
        y = _exact_norm(r, c["kind"]) * v["weight"]
        if v["bias"] is not None:
            y = y + v["bias"]
    out = {"y": y.detach(), "r": r.detach()}
    if train:
        g = _grads((y * s["dy"].double()).sum() + (r * s["dr"].double()).sum(), v)
        out.update(dx=g["x"], dresidual=g["residual"], dweight=g["weight"], dbias=g["bias"],
                   dscale=g["scale"])
    return out


def _exact_after(s, c):
    train = c["mode"] == "train"
    m, d = s["x"].shape
    v = {k: _leaf(s[k]) for k in ("x", "gate", "weight", "bias", "scale")}
    with torch.set_grad_enabled(train):
        gate = v["gate"] * torch.sigmoid(v["gate"])
        p = v["x"] * gate if c["inside"] else v["x"]
        p = _exact_norm(p.view(m, c["groups"], d // c["groups"]), c["kind"]).view(m, d)
        p = p * v["weight"]
        if v["bias"] is not None:
            p = p + v["bias"]
        if not c["inside"]:
            p = p * gate
        res = s["residual"].double() + v["scale"] * p
    out = {"out": res.detach()}
    if train:
        g = _grads((res * s["dout"].double()).sum(), v)
        out.update(dx=g["x"], dgate=g["gate"], dweight=g["weight"], dbias=g["bias"],
                   dscale=g["scale"])
    return out


def _exact_long(s, c):
    if c["mode"] == "step":
        hist = s["history"].clone()
        rows = []
        for i, p in enumerate(s["positions"].tolist()):
            hist[i, :, p] = s["x"][i]
            rows.append((hist[i, :, :p + 1].double() * s["kernel"][:, :p + 1].double().flip(1)).sum(1))
        y = torch.stack(rows) + s["skip"].double() * s["x"].double()
        return {"y": y, "history": hist.double()}
    train = c["mode"] == "train"
    n = c["length"]
    parts = []
    width = max(1, (1 << 25) // (c["batch"] * n))
    for lo in range(0, c["channels"], width):
        q = slice(lo, lo + width)
        v = {"x": _leaf(s["x"][:, q]), "kernel": _leaf(s["kernel"][q]), "skip": _leaf(s["skip"][q])}
        with torch.set_grad_enabled(train):
            prod = torch.fft.rfft(v["x"], 2 * n) * torch.fft.rfft(v["kernel"], 2 * n)
            y = torch.fft.irfft(prod, 2 * n)[..., :n] + v["skip"][:, None] * v["x"]
        p = {"y": y.detach()}
        if train:
            g = _grads((y * s["dy"][:, q].double()).sum(), v)
            p.update(dx=g["x"], dkernel=g["kernel"], dskip=g["skip"])
        parts.append(p)
    axis = {"y": 1, "dx": 1, "dkernel": 0, "dskip": 0}
    return {k: torch.cat([p[k] for p in parts], axis[k]) for k in parts[0]}


_EXACT = {"conv": _exact_conv, "scan": _exact_scan, "before": _exact_before,
          "after": _exact_after, "long": _exact_long}
