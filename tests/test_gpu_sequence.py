"""Sequence operators on the GPU against plain implementations in 64 bits.

Tolerances. Every output is rounded once to its type, which allows
u(type) * |ref| (u = 2^-24, 2^-11, 2^-8). What comes before runs in float32:
its error is counted in units of 2^-24 times the largest reference value of
the tensor, `c` units, with c an upper bound on the roundings between the
inputs and an output (each operator's c is derived where it is set). The terms
of a sum are of the size of the results here (random signs), and a factor of 4
covers sums that cancel.
"""

from __future__ import annotations

import math

import pytest
import torch

from conftest import gpu_available

from ferrum_gpu import capi, sequence as sq

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TYPES = [torch.float32, torch.float16, torch.bfloat16]
F32 = torch.float32


@pytest.fixture(autouse=True, scope="module")
def _gpu():
    if not gpu_available():
        pytest.skip("no B200")


def rnd(seed, *shape, dtype=F32, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to("cuda").to(dtype)


def check(got, ref, c, what=""):
    assert tuple(got.shape) == tuple(ref.shape), what
    if ref.numel() == 0:
        return
    g, r = got.detach().double(), ref.detach().double()
    assert bool(torch.isfinite(g).all()), f"{what}: not finite"
    # float16 results below its normal range are spaced 2^-24 apart
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0.0
    bound = U[got.dtype] * r.abs() + 4 * c * 2.0 ** -24 * r.abs().max() + tiny
    worst = ((g - r).abs() - bound).max().item()
    assert worst <= 0, f"{what}: error {(g - r).abs().max().item():.3e} above its bound by {worst:.3e}"


def dbl(x):
    return None if x is None else x.detach().double().requires_grad_(True)


def silu(x):
    return x * torch.sigmoid(x)


def inside(lengths, b, n):
    if lengths is None:
        return torch.ones(b, n, 1, dtype=torch.bool, device="cuda")
    return (torch.arange(n, device="cuda")[None] < lengths[:, None].long())[:, :, None]


def ends(lengths, b, n):
    return [n] * b if lengths is None else [min(max(int(v), 0), n) for v in lengths]


# ---------------------------------------------------------------- short convolution
# Roundings: K products and sums, bias, then the sigmoid (exponential 2 units,
# sum, quotient 2 units) and two products: K + 16 covers value and slope. A
# parameter's gradient adds the sums over a run of steps and over the runs.

def ref_conv(x, w, bias, act, st, lengths):
    b, n, d = x.shape
    k = w.shape[1]
    keep = inside(lengths, b, n)
    x = torch.where(keep, x, torch.zeros((), dtype=x.dtype, device="cuda"))
    st = torch.zeros(b, k - 1, d, dtype=x.dtype, device="cuda") if st is None else st
    line = torch.cat([st, x], 1)
    p = sum(line[:, j:j + n] * w[:, j] for j in range(k)) + (0 if bias is None else bias)
    y = torch.where(keep, silu(p) if act else p, torch.zeros((), dtype=x.dtype, device="cuda"))
    return y, torch.stack([line[i, e:e + k - 1] for i, e in enumerate(ends(lengths, b, n))])


CONV = [  # batch, length, channels, taps, silu, state, ragged
    (1, 1, 1, 1, False, False, False),
    (2, 1, 33, 4, True, True, False),
    (3, 7, 5, 8, True, False, False),
    (2, 64, 256, 4, True, True, False),
    (2, 65, 257, 3, False, True, True),
    (4, 129, 96, 4, True, True, True),
    (5, 300, 130, 2, True, False, True),
    (3, 257, 1024, 4, True, True, False),
]


def conv_inputs(case, dtype, seed=0):
    b, n, d, k, act, state, ragged = case
    x, dy = rnd(seed, b, n, d, dtype=dtype), rnd(seed + 1, b, n, d, dtype=dtype)
    w, bias = rnd(seed + 2, d, k, std=k ** -0.5), rnd(seed + 3, d)
    st = rnd(seed + 4, b, k - 1, d, dtype=dtype) if state else None
    ln = None
    if ragged:   # empty, full, and beyond both ends of the range (clamped)
        ln = torch.tensor([(0, n, n // 2, n + 5, -3)[i % 5] for i in range(b)],
                          dtype=torch.int32, device="cuda")
        pad = ~inside(ln, b, n).expand(b, n, d)
        x[pad], dy[pad] = float("nan"), float("inf")    # never read
    return x, dy, w, bias, st, ln, "silu" if act else None


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", CONV)
def test_conv(case, dtype):
    x, dy, w, bias, st, ln, act = conv_inputs(case, dtype)
    b, n, d, k = case[:4]
    xd, wd, bd, sd = dbl(x), dbl(w), dbl(bias), dbl(st)
    yr, fr = ref_conv(xd, wd, bd, act, sd, ln)
    y, fin = sq.causal_conv1d(x, w, bias, activation=act, initial_state=st, lengths=ln,
                              return_final_state=True)
    c = k + 16
    check(y, yr, c, "y")
    assert torch.equal(fin.double(), fr.detach())       # copied values
    dfin = rnd(77, *fin.shape, dtype=dtype)
    keep = inside(ln, b, n)
    g = torch.where(keep, dy.double(), torch.zeros((), dtype=torch.float64, device="cuda"))
    leaves = [v for v in (xd, wd, bd, sd) if v is not None]
    ref = torch.autograd.grad((yr * g).sum() + (fr * dfin.double()).sum(), leaves,
                              allow_unused=True)
    got = sq.causal_conv1d_backward(dy, x, w, bias, activation=act, initial_state=st, lengths=ln,
                                    dfinal_state=dfin)
    refx = torch.nan_to_num(ref[0]) if ref[0] is not None else torch.zeros_like(xd)
    check(got.dx, torch.where(keep, refx, torch.zeros((), dtype=torch.float64, device="cuda")),
          2 * c, "dx")
    check(got.dweight, ref[1], c + min(n, 64) + b * (n // 64 + 1), "dweight")
    check(got.dbias, ref[2], c + min(n, 64) + b * (n // 64 + 1), "dbias")
    if st is None:
        assert got.dinitial_state is None
    elif k > 1:
        check(got.dinitial_state, ref[3], 2 * c, "dinitial_state")


@pytest.mark.parametrize("dtype", TYPES)
def test_conv_step_continues_a_prompt(dtype):
    b, n, d, k = 3, 21, 70, 4
    x, w, bias = rnd(1, b, n + 6, d, dtype=dtype), rnd(2, d, k), rnd(3, d)
    whole = sq.causal_conv1d(x, w, bias, activation="silu")
    y, st = sq.causal_conv1d(x[:, :n], w, bias, activation="silu", return_final_state=True)
    assert torch.equal(y, whole[:, :n])
    for t in range(n, n + 6):
        nxt = torch.empty_like(st)
        o = sq.causal_conv1d_step(x[:, t], st, w, bias, activation="silu", next_state=nxt)
        o2 = sq.causal_conv1d_step(x[:, t], st, w, bias, activation="silu")    # in place
        assert torch.equal(o, o2) and torch.equal(st, nxt)
        check(o, ref_conv(dbl(x), dbl(w), dbl(bias), True, None, None)[0][:, t], k + 16, f"step {t}")
        assert torch.equal(st, x[:, t - k + 2:t + 1])


def test_conv_strides_and_out():
    """Slices of a wider projection as input, a slice of a wider array as output."""
    wide = rnd(5, 2, 40, 3 * 48 + 1, dtype=torch.bfloat16)
    x = wide[:, :, 49:97]                    # 2-byte aligned rows
    w = rnd(6, 48, 4)
    host = torch.zeros(2, 40, 100, dtype=torch.bfloat16, device="cuda")
    got = sq.causal_conv1d(x, w, out=host[:, :, 3:51])
    check(got, ref_conv(dbl(x), dbl(w), None, False, None, None)[0], 20)
    assert not host[:, :, :3].any() and not host[:, :, 51:].any()
    with pytest.raises(ValueError, match="contiguous"):
        sq.causal_conv1d(x.transpose(1, 2).contiguous().transpose(1, 2), w)
    with pytest.raises(ValueError, match="one of the inputs"):
        y = x.contiguous()
        sq.causal_conv1d(y, w, out=y)


# ---------------------------------------------------------------- scan
# A state passes through at most n steps. Each multiplies by an exponential
# whose relative error is the unit's (2 units), the product's and its
# argument's (|dt A log2 e| units, below 8 here), and adds a product: 12
# units a step, decaying with the state; 12 n + 16 N bounds value and y's sum.
# Gradients run through the recurrence twice.

def ref_scan(u, delta, A, B, C, D, z, bias, softplus, h, lengths):
    b, n, d = u.shape
    N, G = A.shape[1], B.shape[2]
    zero = torch.zeros((), dtype=torch.float64, device="cuda")
    keep = inside(lengths, b, n)
    s = torch.where(keep, delta if bias is None else delta + bias, zero)
    dt = torch.nn.functional.softplus(s, threshold=60.0) if softplus else s
    u, dt = torch.where(keep, u, zero), torch.where(keep, dt, zero)
    B, C = torch.where(keep[..., None], B, zero), torch.where(keep[..., None], C, zero)
    h = torch.zeros(b, d, N, dtype=torch.float64, device="cuda") if h is None else h
    Bd, Cd = B.repeat_interleave(d // G, 2), C.repeat_interleave(d // G, 2)
    ys = []
    for t in range(n):
        h = torch.exp(dt[:, t, :, None] * A) * h + (dt[:, t] * u[:, t])[..., None] * Bd[:, t]
        ys.append((h * Cd[:, t]).sum(-1))
    y = torch.stack(ys, 1) if n else torch.zeros_like(u)
    if D is not None:
        y = y + D * u
    if z is not None:
        y = y * silu(torch.where(keep, z, zero))
    return torch.where(keep, y, zero), h


SCAN = [  # batch, length, channels, states, groups, full (D, z, bias, softplus, state), ragged
    (1, 1, 1, 1, 1, True, False),
    (2, 1, 40, 16, 1, True, False),
    (1, 2, 64, 16, 2, False, False),
    (2, 63, 33, 8, 1, True, False),
    (2, 64, 64, 16, 1, True, False),
    (2, 65, 48, 16, 2, True, True),
    (3, 130, 66, 13, 3, True, True),
    (1, 300, 32, 32, 1, True, False),
    (5, 97, 20, 16, 1, True, True),
    (1, 193, 70, 64, 2, False, False),
    (1, 1030, 16, 16, 1, True, False),
    (2, 256, 160, 16, 1, False, True),
    # more channels: every split of a channel's steps and states over lanes
    (1, 270, 1100, 16, 1, True, False),
    (2, 140, 1604, 16, 2, True, True),
    (4, 100, 1702, 13, 1, True, True),
    (7, 90, 1800, 16, 1, True, False),
    (1, 135, 1001, 64, 1, True, False),
    (3, 131, 1002, 32, 2, False, True),
    (3, 70, 4100, 8, 1, True, True),
]


def scan_inputs(case, dtype, seed=100):
    b, n, d, N, G, full, ragged = case
    r = lambda i, *s, **k: rnd(seed + i, *s, **k)
    a = dict(u=r(0, b, n, d, dtype=dtype), delta=r(1, b, n, d, dtype=dtype, std=0.5),
             A=-(torch.arange(1, N + 1, device="cuda", dtype=F32) * torch.exp(r(2, d, N, std=0.2))),
             B=r(3, b, n, G, N, dtype=dtype), C=r(4, b, n, G, N, dtype=dtype))
    if full:
        k = dict(D=r(5, d), z=r(6, b, n, d, dtype=dtype), delta_bias=r(7, d, std=0.5) - 2.5,
                 delta_softplus=True)
        h0 = r(8, b, d, N)
    else:
        a["delta"] = (a["delta"].abs() * 0.2).to(dtype)
        k, h0 = dict(D=None, z=None, delta_bias=None, delta_softplus=False), None
    ln = None
    dout = r(9, b, n, d, dtype=dtype)
    if ragged:
        ln = torch.tensor([(0, n, n // 2, n + 5, -3)[i % 5] for i in range(b)],
                          dtype=torch.int32, device="cuda")
        pad = ~inside(ln, b, n)
        for t in (a["u"], a["delta"], k["z"], dout):
            if t is not None:
                t[pad.expand_as(t)] = float("nan")
        a["B"][pad[..., None].expand_as(a["B"])] = float("inf")
        a["C"][pad[..., None].expand_as(a["C"])] = float("nan")
    return a, k, h0, ln, dout


def scan_ref(a, k, h0, ln):
    return ref_scan(a["u"], a["delta"], a["A"], a["B"], a["C"], k["D"], k["z"], k["delta_bias"],
                    k["delta_softplus"], h0, ln)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", SCAN)
def test_scan(case, dtype):
    a, k, h0, ln, dout = scan_inputs(case, dtype)
    b, n, d, N, G = case[:5]
    ad = {i: dbl(v) for i, v in a.items()}
    kd = {i: dbl(v) if isinstance(v, torch.Tensor) else v for i, v in k.items()}
    hd = dbl(h0)
    yr, fr = scan_ref(ad, kd, hd, ln)
    res = sq.selective_scan(**a, **k, initial_state=h0, lengths=ln, save_states=True)
    c = 12 * n + 16 * N
    check(res.out, yr, c, "out")
    check(res.final_state, fr, c, "final_state")
    plain = sq.selective_scan(**a, **k, initial_state=h0, lengths=ln)
    assert plain.states is None
    assert torch.equal(plain.out, res.out) and torch.equal(plain.final_state, res.final_state)
    dfin = rnd(55, b, d, N)
    zero = torch.zeros((), dtype=torch.float64, device="cuda")
    g = torch.where(inside(ln, b, n), dout.double(), zero)
    names = ["u", "delta", "A", "B", "C"] + [i for i in ("D", "z", "delta_bias") if k[i] is not None]
    leaves = [ad.get(i, kd.get(i)) for i in names] + ([hd] if hd is not None else [])
    ref = torch.autograd.grad((yr * g).sum() + (fr * dfin.double()).sum(), leaves, allow_unused=True)
    ref = {i: torch.nan_to_num(v) for i, v in zip(names + ["h0"], ref) if v is not None}
    got = sq.selective_scan_backward(dout, **a, states=res.states, **k, lengths=ln,
                                     dfinal_state=dfin)
    c *= 2
    for name, t in (("u", got.du), ("delta", got.ddelta), ("B", got.dB), ("C", got.dC),
                    ("z", got.dz)):
        if name in ref:
            m = inside(ln, b, n)
            check(t, torch.where(m if t.dim() == 3 else m[..., None], ref[name], zero),
                  c + d, f"d{name}")
    for name, t in (("A", got.dA), ("D", got.dD), ("delta_bias", got.ddelta_bias)):
        if name in ref:
            check(t, ref[name], c + n * b, f"d{name}")
    if hd is not None:
        check(got.dinitial_state, ref["h0"], c, "dinitial_state")
    assert (got.dD is None) == (k["D"] is None) and (got.dz is None) == (k["z"] is None)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,G,d", [(16, 1, 130), (5, 2, 62), (64, 1, 33), (32, 3, 96)])
def test_scan_step_continues_a_prompt(dtype, N, G, d):
    case = (3, 20, d, N, G, True, False)
    a, k, h0, _, _ = scan_inputs(case, dtype)
    cut = lambda t, s: t[:, s] if isinstance(t, torch.Tensor) and t.dim() > 2 else t
    head = {i: cut(v, slice(0, 14)) for i, v in a.items()}
    st = sq.selective_scan(**head, **{i: cut(v, slice(0, 14)) for i, v in k.items()},
                           initial_state=h0).final_state
    yr, fr = scan_ref({i: dbl(v) for i, v in a.items()},
                      {i: dbl(v) if isinstance(v, torch.Tensor) else v for i, v in k.items()},
                      dbl(h0), None)
    for t in range(14, 20):
        at = {i: cut(v, t) for i, v in a.items()}
        kt = {i: cut(v, t) for i, v in k.items()}
        nxt = torch.empty_like(st)
        o = sq.selective_scan_step(**at, state=st, **kt, next_state=nxt)
        o2 = sq.selective_scan_step(**at, state=st, **kt)
        assert torch.equal(o, o2) and torch.equal(st, nxt)
        check(o, yr[:, t], 12 * 20 + 16 * N, f"step {t}")
    check(st, fr, 12 * 20 + 16 * N, "state")


@pytest.mark.parametrize("b,d,N,G", [(83, 4104, 16, 2), (41, 8200, 8, 1), (163, 4096, 5, 1)])
def test_scan_step_of_a_large_batch(b, d, N, G):
    """Batches whose threads take several sequences, the last one short."""
    a, k, h0, _, _ = scan_inputs((b, 1, d, N, G, True, False), torch.bfloat16)
    yr, fr = scan_ref({i: dbl(v) for i, v in a.items()},
                      {i: dbl(v) if isinstance(v, torch.Tensor) else v for i, v in k.items()},
                      dbl(h0), None)
    cut = lambda t: t[:, 0] if isinstance(t, torch.Tensor) and t.dim() > 2 else t
    o = sq.selective_scan_step(**{i: cut(v) for i, v in a.items()}, state=h0,
                               **{i: cut(v) for i, v in k.items()})
    check(o, yr[:, 0], 12 + 16 * N, "out")
    check(h0, fr, 12 + 16 * N, "state")


def test_scan_strides():
    """u and z as halves of one projection, B and C as columns of another; the
    same values give the same bits whatever the strides and alignment."""
    b, n, d, N = 2, 75, 40, 16
    dt = torch.bfloat16
    uz, bc = rnd(1, b, n, 2 * d + 1, dtype=dt), rnd(2, b, n, 2 * N + 5, dtype=dt)
    u, z = uz[..., 1:d + 1], uz[..., d + 1:]
    B, C = bc[..., 5:5 + N], bc[..., 5 + N:]
    delta, A = rnd(3, b, n, d, dtype=dt), -torch.exp(rnd(4, d, N))
    one = sq.selective_scan(u, delta, A, B, C, z=z, delta_softplus=True, save_states=True)
    two = sq.selective_scan(u.contiguous(), delta, A, B.contiguous(), C.contiguous(),
                            z=z.contiguous(), delta_softplus=True)
    assert torch.equal(one.out, two.out)
    yr, _ = ref_scan(dbl(u), dbl(delta), dbl(A), dbl(B)[:, :, None], dbl(C)[:, :, None], None,
                     dbl(z), None, True, None, None)
    check(one.out, yr, 12 * n + 16 * N)
    dout = rnd(6, b, n, d + 3, dtype=dt)[..., 3:]
    g = sq.selective_scan_backward(dout, u, delta, A, B, C, one.states, z=z, delta_softplus=True)
    h = sq.selective_scan_backward(dout.contiguous(), u.contiguous(), delta, A, B.contiguous(),
                                   C.contiguous(), one.states, z=z.contiguous(),
                                   delta_softplus=True)
    for p, q in zip(g, h):
        assert (p is None and q is None) or torch.equal(p, q)


def test_scan_large_steps_and_frozen_states():
    """delta far above and below the softplus's bend; A = 0 keeps the state."""
    b, n, d, N = 1, 70, 8, 4
    u, B, C = rnd(1, b, n, d), rnd(2, b, n, 1, N), rnd(3, b, n, 1, N)
    delta = torch.linspace(-100, 60, n, device="cuda")[None, :, None].expand(b, n, d).contiguous()
    A = torch.zeros(d, N, device="cuda")
    A[:, 1:] = -rnd(4, d, N - 1).abs()
    r = sq.selective_scan(u, delta, A, B, C, delta_softplus=True)
    yr, fr = ref_scan(dbl(u), dbl(delta), dbl(A), dbl(B), dbl(C), None, None, None, True, None, None)
    # exponents reach 60 * |A| log2 e: up to 300 units each
    check(r.out, yr, 400 * n)
    check(r.final_state, fr, 400 * n)


# ---------------------------------------------------------------- norms
# Roundings: the row's sums over D values in float32 (a tree: at most D / 256 +
# 16 units on mean and square), the root and quotient, and a dozen products
# and sums. Column sums run over the rows.

def ref_norm(v, kind, eps, groups=1):
    s = v.shape
    v = v.reshape(s[0], groups, -1)
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    return (v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)).reshape(s)


ROWS = [(1, 1), (3, 7), (5, 64), (33, 257), (2, 1000), (130, 768), (17, 4096), (3, 5001), (2, 20000),
        (3, 6000), (2, 9001)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,d", ROWS)
@pytest.mark.parametrize("kind,parts,res32", [("rms", "rsb", True), ("layer", "rsb", False),
                                              ("rms", "r", True), ("layer", "", False),
                                              ("rms", "s", False)])
def test_norm_before(dtype, m, d, kind, parts, res32):
    if kind == "layer" and d == 1:
        pytest.skip("a single value has no deviation")
    rdt = F32 if res32 else dtype
    x, w = rnd(1, m, d, dtype=dtype), 1 + rnd(2, d, std=0.2)
    res = rnd(3, m, d, dtype=rdt, std=2.0) if "r" in parts else None
    scale = 0.5 + rnd(4, d, std=0.2) if "s" in parts else None
    bias = rnd(5, d) if "b" in parts else None
    xd, wd, rd, sd, bd = dbl(x), dbl(w), dbl(res), dbl(scale), dbl(bias)
    v = (xd if sd is None else xd * sd) + (0 if rd is None else rd)
    y, r = sq.norm_before(x, w, bias, residual=res, scale=scale, kind=kind, eps=1e-5)
    yr = ref_norm(v, kind, 1e-5) * wd + (0 if bd is None else bd)
    c = d / 256 + 48
    check(r, v, 4, "r")
    check(y, yr, c, "y")
    # the backward starts from r as it was stored
    q = r.detach().double().requires_grad_(True)
    yq = ref_norm(q, kind, 1e-5) * wd + (0 if bd is None else bd)
    dy, dr = rnd(6, m, d, dtype=dtype), rnd(7, m, d, dtype=r.dtype)
    leaves = [t for t in (q, wd, bd) if t is not None]
    ref = torch.autograd.grad((yq * dy.double()).sum() + (q * dr.double()).sum(), leaves)
    got = sq.norm_before_backward(dy, r, w, bias, dr=dr, x=x, scale=scale, kind=kind, eps=1e-5)
    check(got.dresidual, ref[0], 2 * c, "dresidual")
    check(got.dx, ref[0] if sd is None else ref[0] * sd, 2 * c, "dx")
    check(got.dweight, ref[1], 2 * c + m, "dweight")
    assert (got.dbias is None) == (bias is None) and (got.dscale is None) == (scale is None)
    if bias is not None:
        check(got.dbias, ref[2], m, "dbias")
    if scale is not None:
        check(got.dscale, (ref[0] * xd).sum(0), 2 * c + m, "dscale")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,d,groups", [(1, 1, 1), (3, 12, 4), (5, 64, 1), (33, 258, 2),
                                        (7, 1000, 8), (130, 768, 1), (9, 4096, 8), (3, 5005, 5),
                                        (2, 20000, 1), (3, 6000, 1), (2, 9001, 1)])
@pytest.mark.parametrize("kind,where,parts", [("rms", "in", "rsb"), ("layer", "out", "rsb"),
                                              ("rms", "out", "r"), ("layer", "none", "s"),
                                              ("layer", "in", "")])
def test_norm_after(dtype, m, d, groups, kind, where, parts):
    if kind == "layer" and d == groups:
        pytest.skip("a single value has no deviation")
    x, w = rnd(1, m, d, dtype=dtype), 1 + rnd(2, d, std=0.2)
    gate = rnd(8, m, d, dtype=dtype) if where != "none" else None
    res = rnd(3, m, d, dtype=F32 if kind == "rms" else dtype) if "r" in parts else None
    scale = 0.5 + rnd(4, d, std=0.2) if "s" in parts else None
    bias = rnd(5, d) if "b" in parts else None
    xd, wd, gd, sd, bd = dbl(x), dbl(w), dbl(gate), dbl(scale), dbl(bias)
    p = ref_norm(xd * silu(gd) if where == "in" else xd, kind, 1e-5, groups) * wd
    p = p + (0 if bd is None else bd)
    if where == "out":
        p = p * silu(gd)
    yr = (p if sd is None else p * sd) + (0 if res is None else res.double())
    kw = dict(gate=gate, gate_inside=where == "in", scale=scale, groups=groups, kind=kind, eps=1e-5)
    y = sq.norm_after(x, w, bias, residual=res, **kw)
    c = d / groups / 256 + 64
    check(y, yr, c, "y")
    dout = rnd(6, m, d, dtype=dtype)
    leaves = {"x": xd, "gate": gd, "weight": wd, "bias": bd, "scale": sd}
    live = {i: v for i, v in leaves.items() if v is not None}
    ref = dict(zip(live, torch.autograd.grad((yr * dout.double()).sum(), list(live.values()))))
    got = sq.norm_after_backward(dout, x, w, bias, **kw)
    check(got.dx, ref["x"], 2 * c, "dx")
    for name, t, cc in (("gate", got.dgate, 2 * c), ("weight", got.dweight, 2 * c + m),
                        ("bias", got.dbias, 2 * c + m), ("scale", got.dscale, 2 * c + m)):
        assert (t is None) == (name not in live)
        if t is not None:
            check(t, ref[name], cc, f"d{name}")


def test_norm_rows_of_zeros_and_strides():
    x = torch.zeros(3, 40, device="cuda")
    x[1] = 1e-20
    y, r = sq.norm_before(x, torch.ones(40, device="cuda"))
    assert torch.equal(r, x) and bool(torch.isfinite(y).all()) and not y[0].any()
    g = sq.norm_before_backward(torch.ones_like(x), r, torch.ones(40, device="cuda"))
    assert bool(torch.isfinite(g.dx).all())
    wide = rnd(1, 6, 5, 101, dtype=torch.bfloat16)
    xs = wide[..., 1:41]
    w = torch.ones(40, device="cuda")
    assert torch.equal(sq.norm_before(xs, w)[0], sq.norm_before(xs.contiguous(), w)[0])
    host = torch.zeros(6, 5, 50, dtype=torch.bfloat16, device="cuda")
    got = sq.norm_after(xs, w, gate=wide[..., 45:85], out=host[..., 7:47])
    want = sq.norm_after(xs.contiguous(), w, gate=wide[..., 45:85].contiguous())
    assert torch.equal(got, want) and not host[..., :7].any() and not host[..., 47:].any()
    # one row's infinity stays in its row
    x = rnd(2, 4, 300)
    clean = sq.norm_before(x, torch.ones(300, device="cuda"))[0]
    x[2, 5] = float("inf")
    bad = sq.norm_before(x, torch.ones(300, device="cuda"))[0]
    assert torch.equal(bad[[0, 1, 3]], clean[[0, 1, 3]]) and not bool(torch.isfinite(bad[2]).all())


# ---------------------------------------------------------------- long convolution
# By transforms: a radix-16 or 32 stage adds about 8 units relative to the
# largest value of its array in the root-mean-square sense; forward, product
# and inverse have 2 log2 N / 4 + 2 stages, so 16 log2 N units; sums over the
# batch (dkernel) add b. By definition (short rows): one unit per tap.

def ref_long(x, k, skip):
    n = x.shape[-1]
    m = max(2, 2 * n)
    y = torch.fft.irfft(torch.fft.rfft(x, m) * torch.fft.rfft(k, m), m)[..., :n]
    return y if skip is None else y + skip[:, None] * x


LONG = [(1, 1, 1, 1), (2, 3, 2, 2), (3, 5, 17, 17), (2, 4, 64, 30), (1, 3, 100, 100),
        (3, 7, 129, 129), (2, 5, 255, 200), (1, 2, 256, 256), (3, 9, 500, 500), (2, 3, 513, 513), (3, 4, 1000, 1000),
        (2, 2, 2048, 2048), (1, 3, 4095, 1), (2, 2, 4096, 4096), (3, 2, 5000, 4000),
        (1, 2, 8193, 8193), (2, 1, 16384, 16384), (1, 2, 16385, 16385), (1, 1, 40000, 40000)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,d,n,taps", LONG)
def test_long_conv(dtype, b, d, n, taps):
    x, dy = rnd(1, b, d, n, dtype=dtype), rnd(2, b, d, n, dtype=dtype)
    k, skip = rnd(3, d, taps, std=taps ** -0.5), rnd(4, d)
    c = 16 * math.log2(2 * n + 2) + min(n, 64)
    for sk in (skip, None):
        xd, kd, sd = dbl(x), dbl(k), dbl(sk)
        yr = ref_long(xd, kd, sd)
        check(sq.long_conv(x, k, sk), yr, c, "y")
        leaves = [t for t in (xd, kd, sd) if t is not None]
        ref = torch.autograd.grad((yr * dy.double()).sum(), leaves)
        got = sq.long_conv_backward(dy, x, k, sk)
        check(got.dx, ref[0], c, "dx")
        check(got.dkernel, ref[1], c + b, "dkernel")
        if sk is not None:
            check(got.dskip, ref[2], c + b + n / 32, "dskip")
        else:
            assert got.dskip is None


@pytest.mark.parametrize("n", [40, 700])
def test_long_conv_channel_last_and_slices(n):
    dt = torch.bfloat16
    wide = rnd(1, 3, n, 21, dtype=dt)
    x = wide[..., 2:13].transpose(1, 2)             # (3, 11, n), steps of 21
    k, skip = rnd(2, 11, n, std=n ** -0.5), rnd(3, 11)
    y = sq.long_conv(x, k, skip)
    assert torch.equal(y, sq.long_conv(x.contiguous(), k, skip))
    host = torch.zeros(3, n, 16, dtype=dt, device="cuda")
    sq.long_conv(x, k, skip, out=host[..., 1:12].transpose(1, 2))
    assert torch.equal(host[..., 1:12].transpose(1, 2), y) and not host[..., 12:].any()
    dy = torch.ones((), dtype=dt, device="cuda").expand(3, 11, n)       # every stride 0
    g, h = sq.long_conv_backward(dy, x, k, skip), sq.long_conv_backward(
        dy.contiguous(), x.contiguous(), k, skip)
    for p, q in zip(g, h):
        assert torch.equal(p, q)
    odd = rnd(4, 3, 11, n + 1, dtype=dt)[..., 1:]   # rows at odd addresses
    assert torch.equal(sq.long_conv(odd, k), sq.long_conv(odd.contiguous(), k))


def test_long_conv_keeps_rows_apart():
    x, k = rnd(1, 4, 3, 900), rnd(2, 3, 900, std=0.03)
    clean = sq.long_conv(x, k)
    x[2, 1, 17] = float("nan")
    bad = sq.long_conv(x, k)
    row = torch.ones(4, 3, dtype=torch.bool, device="cuda")
    row[2, 1] = False
    assert torch.equal(bad[row], clean[row]) and bool(torch.isnan(bad[2, 1, 17:]).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap,taps", [(1, 1), (5, 3), (100, 100), (1030, 900)])
def test_long_conv_step(dtype, cap, taps):
    b, d = 5, 9
    hist = rnd(1, b, d, cap, dtype=dtype)
    x, k, skip = rnd(2, b, d, dtype=dtype), rnd(3, d, taps, std=taps ** -0.5), rnd(4, d)
    pos = torch.tensor([0, cap - 1, cap // 2, -1, cap], dtype=torch.int32, device="cuda")
    keep = hist.clone()
    y = sq.long_conv_step(x, hist, pos, k, skip)
    for i, p in enumerate([0, cap - 1, cap // 2]):
        line = torch.cat([keep[i, :, :p], x[i][:, None]], 1)
        full = ref_long(line[None].double(), k[:, :p + 1].double(), skip.double())[0, :, -1]
        check(y[i], full, 64 + min(p, 64), f"row {i}")
        keep[i, :, p] = x[i]
    assert not y[3:].any()
    assert torch.equal(hist, keep)


# ---------------------------------------------------------------- differences
# loss(p) = sum of w * output in 64 bits. Its central difference over 2 e in a
# direction v differs from <grad, v> by e^2 / 6 times the third derivative
# (of the size of the derivative itself here) and by the float32 roundings of
# the outputs, c 2^-24 of their size each, at random: times sqrt(outputs) / e.

def directional(loss, inputs, grads, c, outputs, size, seed=900):
    e = 2.0 ** -6
    vs = [rnd(seed + i, *t.shape) for i, t in enumerate(inputs)]
    up = loss(*[t + e * v for t, v in zip(inputs, vs)])
    down = loss(*[t - e * v for t, v in zip(inputs, vs)])
    diff = (up - down).item() / (2 * e)
    want = sum((g.double() * v.double()).sum().item() for g, v in zip(grads, vs))
    total = math.sqrt(sum((g.double() ** 2).sum().item() for g in grads))
    bound = 64 * e * e * total + 4 * c * 2.0 ** -24 * size * math.sqrt(outputs) / e
    assert abs(diff - want) <= bound, (diff, want, bound)


def test_gradients_against_differences():
    b, n, d, N = 2, 70, 24, 16
    w = rnd(50, b, n, d)
    ws = rnd(51, b, d, N)
    a, k, h0, _, _ = scan_inputs((b, n, d, N, 1, True, False), F32)

    def scan(u, delta, A, B, C, D, z, bias, h):
        r = sq.selective_scan(u, delta, A, B, C, D=D, z=z, delta_bias=bias, delta_softplus=True,
                              initial_state=h)
        return (r.out.double() * w.double()).sum() + (r.final_state.double() * ws.double()).sum()

    st = sq.selective_scan(**a, **k, initial_state=h0, save_states=True).states
    g = sq.selective_scan_backward(w, **a, states=st, **k, dfinal_state=ws)
    ins = [a[i] for i in ("u", "delta", "A", "B", "C")] + [k["D"], k["z"], k["delta_bias"], h0]
    gs = [g.du, g.ddelta, g.dA, g.dB, g.dC, g.dD, g.dz, g.ddelta_bias, g.dinitial_state]
    for i in range(len(ins)):       # one argument at a time
        directional(lambda t: scan(*[t if j == i else v for j, v in enumerate(ins)]), [ins[i]],
                    [gs[i]], 12 * n + 16 * N, b * n * d, 8.0, 900 + 20 * i)

    x, cw, cb, cs = rnd(1, b, n, d), rnd(2, d, 4), rnd(3, d), rnd(4, b, 3, d)
    g = sq.causal_conv1d_backward(w, x, cw, cb, activation="silu", initial_state=cs)

    def conv(x, cw, cb, cs):
        y = sq.causal_conv1d(x, cw, cb, activation="silu", initial_state=cs)
        return (y.double() * w.double()).sum()

    directional(conv, [x, cw, cb, cs], [g.dx, g.dweight, g.dbias, g.dinitial_state], 20,
                b * n * d, 8.0)

    gate, nw, nb, sc = rnd(5, b * n, d), rnd(6, d), rnd(7, d), rnd(8, d)
    xm, wm = x.view(-1, d), w.view(-1, d)
    for where in (True, False):
        for kind in ("rms", "layer"):
            kw = dict(gate_inside=where, groups=2, kind=kind)
            g = sq.norm_after_backward(wm, xm, nw, nb, gate=gate, scale=sc, **kw)
            directional(lambda x, gate, nw, nb, sc: (sq.norm_after(
                x, nw, nb, gate=gate, scale=sc, **kw).double() * wm.double()).sum(),
                [xm, gate, nw, nb, sc], [g.dx, g.dgate, g.dweight, g.dbias, g.dscale], 80,
                b * n * d, 8.0)

    dr = rnd(9, b * n, d)
    y, r = sq.norm_before(xm, nw, nb, residual=gate, scale=sc, kind="layer")
    g = sq.norm_before_backward(wm, r, nw, nb, dr=dr, x=xm, scale=sc, kind="layer")

    def before(x, res, nw, nb, sc):
        y, r = sq.norm_before(x, nw, nb, residual=res, scale=sc, kind="layer")
        return (y.double() * wm.double()).sum() + (r.double() * dr.double()).sum()

    directional(before, [xm, gate, nw, nb, sc], [g.dx, g.dresidual, g.dweight, g.dbias, g.dscale],
                80, 2 * b * n * d, 8.0)

    xl, kl, sl = rnd(10, 2, 6, 500), rnd(11, 6, 500, std=0.05), rnd(12, 6)
    wl = rnd(13, 2, 6, 500)
    g = sq.long_conv_backward(wl, xl, kl, sl)
    directional(lambda x, k, s: (sq.long_conv(x, k, s).double() * wl.double()).sum(),
                [xl, kl, sl], [g.dx, g.dkernel, g.dskip], 250, 6000, 8.0)


# ---------------------------------------------------------------- empty calls, streams, refusals

def test_empty_sizes():
    dt = torch.bfloat16
    for b, n, d in ((0, 5, 4), (2, 0, 4), (2, 5, 0)):
        x = torch.zeros(b, n, d, dtype=dt, device="cuda")
        st = rnd(1, b, 3, d, dtype=dt)
        y, fin = sq.causal_conv1d(x, torch.ones(d, 4, device="cuda"), initial_state=st,
                                  return_final_state=True)
        assert y.shape == x.shape
        if n == 0:
            assert torch.equal(fin, st)         # an empty prompt keeps its state
        g = sq.causal_conv1d_backward(x, x, torch.ones(d, 4, device="cuda"),
                                      torch.ones(d, device="cuda"))
        if not (b and n and d):
            assert not g.dweight.any() and not g.dbias.any()
        A, bc = -torch.ones(d, 4, device="cuda"), torch.zeros(b, n, 4, dtype=dt, device="cuda")
        h0 = rnd(2, b, d, 4)
        r = sq.selective_scan(x, x, A, bc, bc, initial_state=h0, save_states=True)
        if n == 0:
            assert torch.equal(r.final_state, h0)
        dfin = rnd(3, b, d, 4)
        g = sq.selective_scan_backward(x, x, x, A, bc, bc, r.states, dfinal_state=dfin)
        assert not g.dA.any()
        if n == 0:
            assert torch.equal(g.dinitial_state, dfin)
        m = x.reshape(-1, d) if d else x.reshape(10, 0)
        w = torch.ones(d, device="cuda")
        sq.norm_before(m, w), sq.norm_after(m, w)
        assert not sq.norm_before_backward(m, m, w).dweight.any()
        assert not sq.norm_after_backward(m, m, w).dweight.any()
        k = torch.zeros(n, min(d, 1), device="cuda")
        assert sq.long_conv(x, k).shape == x.shape
        assert not sq.long_conv_backward(x, x, k).dkernel.any()


def test_other_stream_and_determinism():
    a, k, h0, _, dout = scan_inputs((2, 200, 96, 16, 1, True, False), torch.bfloat16)
    want = sq.selective_scan(**a, **k, initial_state=h0, save_states=True)
    gw = sq.selective_scan_backward(dout, **a, states=want.states, **k)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for stream in (s, s.cuda_stream):
        for _ in range(5):
            got = sq.selective_scan(**a, **k, initial_state=h0, save_states=True, stream=stream)
            gg = sq.selective_scan_backward(dout, **a, states=got.states, **k, stream=stream)
            s.synchronize()
            assert torch.equal(got.out, want.out)
            for p, q in zip(gg, gw):
                assert torch.equal(p, q)


def test_graph_capture_of_a_decode_step():
    b, d, N = 4, 64, 16
    dt = torch.bfloat16
    x, cst, w = rnd(1, b, d, dtype=dt), rnd(2, b, 3, d, dtype=dt), rnd(3, d, 4)
    sst, A, bc = rnd(4, b, d, N), -torch.exp(rnd(5, d, N)), rnd(6, b, N, dtype=dt)

    def step():
        u = sq.causal_conv1d_step(x, cst, w, activation="silu")
        return sq.selective_scan_step(u, x, A, bc, bc, sst, delta_softplus=True)

    keep = cst.clone(), sst.clone()
    want = [step().clone() for _ in range(3)]
    cst.copy_(keep[0]), sst.copy_(keep[1])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = step()
    for i in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i])


def test_offsets_beyond_32_bits():
    """Arrays of more than 2^31 values: their last part equals a call on that
    part alone. Steps are cut at a multiple of every internal piece length, so
    the same arithmetic runs and the bits agree."""
    dt = torch.bfloat16
    n, d, cut = (1 << 20) + 40, 2056, 1 << 20
    assert n * d > 2 ** 31
    x = torch.empty(1, n, d, dtype=dt, device="cuda").normal_()
    tail = x[:, cut:].contiguous()
    w = rnd(1, d, 4)
    y = sq.causal_conv1d(x, w, activation="silu")
    st = x[:, cut - 3:cut].contiguous()
    assert torch.equal(y[:, cut:], sq.causal_conv1d(tail, w, activation="silu", initial_state=st))
    g = sq.causal_conv1d_backward(y, x, w, activation="silu")
    h = sq.causal_conv1d_backward(y[:, cut:].contiguous(), tail, w, activation="silu",
                                  initial_state=st)
    assert torch.equal(g.dx[:, cut:], h.dx)
    del g, h
    A, B = -rnd(2, d, 8).abs(), rnd(3, 1, n, 8, dtype=dt)
    one = sq.selective_scan(x, y, A, B, B, delta_softplus=True, save_states=True)
    at = one.states[:, cut // sq.SAVE_STEPS].clone()
    two = sq.selective_scan(tail, y[:, cut:], A, B[:, cut:], B[:, cut:], delta_softplus=True,
                            initial_state=at, save_states=True)
    check(one.out[:, cut:], two.out.double(), 12 * 40)
    check(one.final_state, two.final_state.double(), 12 * 40)
    g = sq.selective_scan_backward(y, x, y, A, B, B, one.states, delta_softplus=True)
    h = sq.selective_scan_backward(y[:, cut:], tail, y[:, cut:], A, B[:, cut:], B[:, cut:],
                                   two.states, delta_softplus=True)
    check(g.du[:, cut:], h.du.double(), 24 * 40 + d)
    check(g.dB[:, cut:], h.dB.double(), 24 * 40 + d)
    del one, two, g, h
    m, wt = x[0], rnd(4, d)
    yb, r = sq.norm_before(m, wt, residual=y[0])
    yt, rt = sq.norm_before(m[cut:], wt, residual=y[0, cut:])
    assert torch.equal(yb[cut:], yt) and torch.equal(r[cut:], rt)
    assert torch.equal(sq.norm_before_backward(yb, r, wt).dx[cut:],
                       sq.norm_before_backward(yt, rt, wt).dx)
    del yb, r
    assert torch.equal(sq.norm_after(m, wt, gate=y[0], groups=8)[cut:],
                       sq.norm_after(m[cut:], wt, gate=y[0, cut:], groups=8))
    assert torch.equal(sq.norm_after_backward(y[0], m, wt, gate=y[0], groups=8).dgate[cut:],
                       sq.norm_after_backward(y[0, cut:], m[cut:], wt, gate=y[0, cut:], groups=8).dgate)
    del x, y, m
    rows, length = 1 << 16, 1 << 15
    x = torch.empty(rows + 8, 1, length, dtype=dt, device="cuda").normal_()
    assert x.numel() > 2 ** 31
    pos = torch.full((rows + 8,), length - 1, dtype=torch.int32, device="cuda")
    k = rnd(5, 1, length, std=length ** -0.5)
    last = x[-8:].clone()
    v = rnd(6, rows + 8, 1, dtype=dt)
    y = sq.long_conv_step(v, x, pos, k)
    assert torch.equal(y[-8:], sq.long_conv_step(v[-8:], last, pos[-8:], k))
    assert torch.equal(x[-8:], last)
    x = x.view(-1, 1, 4096)
    assert torch.equal(sq.long_conv(x, k[:, :4096].contiguous())[-8:],
                       sq.long_conv(x[-8:], k[:, :4096].contiguous()))


def test_refusals():
    x = rnd(1, 2, 6, 8)
    w4 = rnd(2, 8, 4)
    bad = pytest.raises(ValueError)
    with bad:
        sq.causal_conv1d(x.double(), w4)
    with bad:
        sq.causal_conv1d(x, rnd(2, 8, 9))               # taps
    with bad:
        sq.causal_conv1d(x, rnd(2, 7, 4))
    with bad:
        sq.causal_conv1d(x, w4.to(torch.bfloat16))
    with bad:
        sq.causal_conv1d(x, w4, activation="gelu")
    with bad:
        sq.causal_conv1d(x, w4, initial_state=rnd(3, 2, 4, 8))
    with bad:
        sq.causal_conv1d(x, w4, lengths=torch.tensor([3, 4], device="cuda"))     # int64
    with bad:
        sq.causal_conv1d(x, w4, out=torch.empty(2, 6, 1, device="cuda").expand(2, 6, 8))
    with bad:
        sq.causal_conv1d_step(x[:, 0], None, w4)
    A, B = -torch.ones(8, 4, device="cuda"), rnd(4, 2, 6, 4)
    with bad:
        sq.selective_scan(x, x, -torch.ones(8, 65, device="cuda"), B, B)
    with bad:
        sq.selective_scan(x, x, A, rnd(4, 2, 6, 3, 4), rnd(4, 2, 6, 3, 4))       # 3 groups of 8
    with bad:
        sq.selective_scan(x, x, A, B, rnd(4, 2, 5, 4))
    with bad:
        sq.selective_scan(x, x.to(torch.float16), A, B, B)
    with bad:
        sq.selective_scan_backward(x, x, x, A, B, B, None)
    with bad:
        sq.selective_scan_backward(x, x, x, A, B, B, rnd(5, 2, 2, 8, 4))
    with bad:
        sq.norm_before(x, torch.ones(7, device="cuda"))
    with bad:
        sq.norm_before(x, torch.ones(8, device="cuda"), kind="batch")
    with bad:
        sq.norm_before(x, torch.ones(8, device="cuda"), eps=-1.0)
    with bad:
        sq.norm_before(x, torch.ones(8, device="cuda"), residual=x.to(torch.float16))
    with bad:
        sq.norm_after(x, torch.ones(8, device="cuda"), groups=3)
    with bad:
        sq.norm_before(x.transpose(0, 1), torch.ones(8, device="cuda"))
    with bad:
        sq.norm_before_backward(x, x, torch.ones(8, device="cuda"),
                                scale=torch.ones(8, device="cuda"))              # x missing
    with bad:
        sq.long_conv(x, rnd(6, 6, 9))                   # more taps than steps
    with bad:
        sq.long_conv(x, rnd(6, 5, 8))
    with bad:
        sq.long_conv_step(x[:, 0], rnd(7, 2, 8, 5), torch.zeros(2, device="cuda"), rnd(6, 8, 5))
    # the C entries refuse what a C caller can get wrong
    h = capi.DeviceHandle(0)
    args = capi.ConvArgs(struct_size=1)
    assert capi.lib().ferrum_causal_conv1d(h.ptr, args, None) == capi.FERRUM_ERR_INVALID_ARG
    assert "struct_size" in capi.last_error()
    assert capi.lib().ferrum_causal_conv1d(h.ptr, None, None) == capi.FERRUM_ERR_INVALID_ARG
    import ctypes
    args = capi.ConvArgs(struct_size=ctypes.sizeof(capi.ConvArgs), taps=4, batch=1 << 40,
                       length=1 << 20, channels=1 << 20)
    assert capi.lib().ferrum_causal_conv1d(h.ptr, args, None) == capi.FERRUM_ERR_INVALID_ARG
    args = capi.ConvArgs(struct_size=ctypes.sizeof(capi.ConvArgs), taps=4, batch=1, length=1, channels=1)
    assert capi.lib().ferrum_causal_conv1d(h.ptr, args, None) == capi.FERRUM_ERR_INVALID_ARG
    assert "weight is NULL" in capi.last_error()
    h.close()
