"""Sequence operators on the GPU at the ends of their domain: growing and
vanishing states, infinities, small results in relative terms, streams,
arguments of other libraries and arrays that share memory.

Tolerances are counted in units of 2^-24 (float32 roundings), with the count
derived at each test.
"""

from __future__ import annotations

import ctypes

import pytest
import torch

from conftest import gpu_available

from ferrum_gpu import capi, sequence as sq

pytestmark = pytest.mark.gpu

F32 = torch.float32
UNIT = 2.0 ** -24


@pytest.fixture(autouse=True, scope="module")
def _gpu():
    if not gpu_available():
        pytest.skip("no B200")


def rnd(seed, *shape, dtype=F32, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to("cuda").to(dtype)


def full(value, *shape, dtype=F32):
    return torch.full(shape, value, dtype=dtype, device="cuda")


# Batches and channels for every split of a channel's steps and states over
# lanes and warps: 4, 8, 16 lanes, then 2 and 4 warps of 16 (4 take more than
# 8 states).
SPLITS = [(3, 4100), (6, 1001), (3, 1002), (1, 1001), (1, 40)]


# ---------------------------------------------------------------- growing states

def grown(u, dt, A, B, C, h):
    """The recurrence in 64 bits, for constant dt and one group."""
    u, A, B, C, h = (t.double() for t in (u, A, B, C, h))
    a, ys = torch.exp(dt * A), [torch.zeros_like(u[:, 0])]
    for t in range(u.shape[1]):
        h = a * h + (dt * u[:, t])[..., None] * B[:, t, None]
        ys.append((h * C[:, t, None]).sum(-1))
    return torch.stack(ys[1:] or ys, 1), h


@pytest.mark.parametrize("n,rate", [(112, 1.45), (56, 2.9), (28, 5.8)])
@pytest.mark.parametrize("N", [16, 8])
@pytest.mark.parametrize("b,d", SPLITS)
def test_scan_of_growing_states(b, d, N, n, rate):
    """Factors above 1, whose product over some lanes' steps (64, 32, 16 of
    them) passes the largest float32 while the state in front is zero or small:
    e^162 in all, from 1e-37 to 3e33."""
    delta, A = full(1.0, b, n, d), full(rate, d, N)
    B, C = rnd(1, b, n, N).abs(), rnd(2, b, n, N).abs()
    late = torch.zeros(b, n, d, device="cuda")
    tail = int(30 / rate)                            # e^30 behind the first input
    late[:, -tail:] = rnd(3, b, tail, d).abs() + 0.1
    for u, h0 in ((late, full(0.0, b, d, N)), (late * 0, full(1e-37, b, d, N))):
        yr, hr = grown(u, 1.0, A, B, C, h0)
        r = sq.selective_scan(u, delta, A, B, C, initial_state=h0, save_states=True)
        # Every term is positive, so nothing cancels. Units: 8 for a step's
        # exponential, product and sum; one for each nat of the exponents
        # (162) in A log2 e, in a step's product, and twice in a sum of steps.
        tol = (8 * n + 4 * 162 + N) * UNIT
        assert bool(torch.isfinite(r.final_state).all())
        assert ((r.final_state - hr).abs() <= tol * hr).all()
        assert ((r.out - yr).abs() <= tol * yr).all()
        at = (n - 1) // 16                           # the last state saved
        mid = grown(u[:, :16 * at], 1.0, A, B[:, :16 * at], C[:, :16 * at], h0)[1]
        assert ((r.states[:, at] - mid).abs() <= tol * mid).all()


@pytest.mark.parametrize("b,d", SPLITS)
def test_scan_of_states_that_grow_by_negative_steps(b, d):
    """dt A and dt u are the same for -dt, -A, -u: so are the results, to the bit."""
    n, N, rate = 112, 16, 1.45
    B, C, h0 = rnd(1, b, n, N), rnd(2, b, n, N), rnd(3, b, d, N, std=1e-37)
    u, dt = rnd(4, b, n, d, std=1e-37), full(1.0, b, n, d)
    dt[:, ::7] = -0.5                                # some factors below 1 too
    A = full(rate, d, N)
    p = sq.selective_scan(u, dt, A, B, C, initial_state=h0, save_states=True)
    q = sq.selective_scan(-u, -dt, -A, B, C, initial_state=h0, save_states=True)
    assert bool(torch.isfinite(p.final_state).all())
    for x, y in zip(p, q):
        assert torch.equal(x, y)


@pytest.mark.parametrize("n", [5, 64, 150])
@pytest.mark.parametrize("b,d", SPLITS)
def test_scan_states_that_forget_at_once(b, d, n):
    """A = -inf: exp(dt A) = 0 at every step, whatever follows the sequence's
    end inside the last piece."""
    N = 16
    A = -rnd(1, d, N).abs()
    A[:, ::2] = -float("inf")
    u, delta = rnd(2, b, n, d), rnd(3, b, n, d).abs() + 0.1
    B, C = rnd(4, b, n, N), rnd(5, b, n, N)
    h0 = rnd(6, b, d, N)
    r = sq.selective_scan(u, delta, A, B, C, initial_state=h0, save_states=True)
    g = sq.selective_scan_backward(u, u, delta, A, B, C, r.states)
    for t in (r.out, r.final_state, g.du, g.ddelta, g.dA, g.dB, g.dC, g.dinitial_state):
        assert bool(torch.isfinite(t).all())
    last = delta[:, -1].double() * u[:, -1].double()
    want = last[..., None] * B[:, -1, None, ::2].double()
    # two products
    assert not g.dinitial_state[..., ::2].any()
    assert ((r.final_state[..., ::2] - want).abs() <= 4 * UNIT * want.abs()).all()


def test_scan_gradients_are_zero_behind_a_sequence():
    """Whatever the states and the final state's gradient hold."""
    b, n, d, N = 3, 40, 33, 16
    lengths = torch.tensor([5, 0, 21], dtype=torch.int32, device="cuda")
    u, delta, z, dout = (rnd(i, b, n, d) for i in range(4))
    B, C, A = rnd(5, b, n, N), rnd(6, b, n, N), -rnd(7, d, N).abs()
    dfin = h0 = full(float("inf"), b, d, N)
    r = sq.selective_scan(u, delta, A, B, C, z=z, delta_softplus=True, lengths=lengths,
                          initial_state=h0, save_states=True)
    g = sq.selective_scan_backward(dout, u, delta, A, B, C, r.states, z=z, delta_softplus=True,
                                   lengths=lengths, dfinal_state=dfin)
    for i, ln in enumerate((5, 0, 21)):
        for t in (r.out, g.du, g.ddelta, g.dz, g.dB, g.dC):
            assert not t[i, ln:].any()


# ---------------------------------------------------------------- small results

def test_softplus_keeps_its_relative_accuracy():
    """out = dt = softplus(delta) for one step of u = B = C = 1 from a zero
    state. Units: the exponential 4 (2 in its last place), its argument's
    correction 1, the polynomial 3, its products and the sum 3; 12 in all. In
    the gradient ddelta = sigmoid(delta): the exponential 5, the quotient 2 and
    products 3."""
    x = torch.linspace(-87, 30, 20001, device="cuda")
    d = x.numel()
    one, A = full(1.0, 1, 1, d), full(0.0, d, 1)
    bc = full(1.0, 1, 1, 1)
    want = torch.nn.functional.softplus(x.double(), threshold=100.0)
    tol = 12 * UNIT * want
    r = sq.selective_scan(one, x[None, None], A, bc, bc, delta_softplus=True, save_states=True)
    assert ((r.out[0, 0] - want).abs() <= tol).all()
    assert ((r.final_state[0, :, 0] - want).abs() <= tol).all()
    state = full(0.0, 1, d, 1)
    out = sq.selective_scan_step(one[0], x[None], A, bc[0], bc[0], state, delta_softplus=True)
    assert ((out[0] - want).abs() <= tol).all()
    g = sq.selective_scan_backward(one, one, x[None, None], A, bc, bc, r.states,
                                   delta_softplus=True)
    assert ((g.du[0, 0] - want).abs() <= tol).all()
    slope = torch.sigmoid(x.double())
    assert ((g.ddelta[0, 0] - slope).abs() <= 10 * UNIT * slope).all()
    ends = torch.tensor([float("inf"), -float("inf"), float("nan"), -200.0], device="cuda")
    bc = full(1.0, 1, 1, 8)
    r = sq.selective_scan(one[..., :4], ends[None, None], full(-1.0, 4, 8), bc, bc,
                          delta_softplus=True)
    got = r.out[0, 0].tolist()
    assert got[0] == float("inf") and got[1] == 0 and got[2] != got[2] and got[3] == 0


# ---------------------------------------------------------------- long sequences
# A state's error is made anew by each step and decays with it. Per step: the
# exponential 4 units (2 in its last place), its argument |dt A log2 e| <= 2
# twice, product and sum 3: 12 units of the state, so 12 / (1 - a) at most, with
# a the largest factor exp(dt A). Terms are of the size of the results (random
# signs); a factor of 4 covers the sums that cancel, and every error is
# measured against the largest value of its own channel.

LONG = [(1, 1030, 40, 16), (2, 517, 130, 16), (1, 300, 1001, 13), (1, 2049, 33, 32),
        (3, 260, 4100, 8), (6, 150, 1001, 16), (1, 700, 20, 64)]


@pytest.mark.parametrize("b,n,d,N", LONG)
def test_long_scans_keep_float32_accuracy(b, n, d, N):
    u, z, dout = rnd(1, b, n, d), rnd(2, b, n, d), rnd(3, b, n, d)
    delta = rnd(4, b, n, d, std=0.3).abs().clamp(0.05, 1.0)
    A = -(1 + rnd(5, d, N).abs().clamp(max=1.0))       # 1 <= -A <= 2, a <= e^-0.05
    B, C, D, h0 = rnd(6, b, n, N), rnd(7, b, n, N), rnd(8, d), rnd(9, b, d, N)
    leaves = [t.double().requires_grad_(True) for t in (u, delta, A, B, C, D, z, h0)]
    ud, dd, Ad, Bd, Cd, Dd, zd, h = leaves
    ys = []
    for t in range(n):
        h = torch.exp(dd[:, t, :, None] * Ad) * h + (dd[:, t] * ud[:, t])[..., None] * Bd[:, t, None]
        ys.append((h * Cd[:, t, None]).sum(-1))
    out = (torch.stack(ys, 1) + Dd * ud) * zd * torch.sigmoid(zd)
    c = 12 / (1 - torch.exp(torch.tensor(-0.05)).item()) + N + 16

    def close(got, ref, units, dims, what):
        top = ref.abs().amax(dims, keepdim=True)
        worst = ((got - ref).abs() / top).max().item() / UNIT
        assert worst <= 4 * units, f"{what}: {worst:.0f} units above {4 * units:.0f}"

    k = dict(D=D, z=z)
    r = sq.selective_scan(u, delta, A, B, C, initial_state=h0, save_states=True, **k)
    close(r.out, out.detach(), c, 1, "out")
    close(r.final_state, h.detach(), c, 2, "final_state")
    ref = torch.autograd.grad((out * dout.double()).sum(), leaves)
    g = sq.selective_scan_backward(dout, u, delta, A, B, C, r.states, **k)
    # the gradient's recurrence decays alike, on states with errors of their own
    for got, want, units, dims, what in (
            (g.du, ref[0], 2 * c, 1, "du"), (g.ddelta, ref[1], 2 * c + N, 1, "ddelta"),
            (g.dB, ref[3], 2 * c + d ** 0.5, 1, "dB"), (g.dC, ref[4], c + d ** 0.5, 1, "dC"),
            (g.dz, ref[6], c, 1, "dz"), (g.dinitial_state, ref[7], 2 * c, 2, "dinitial_state"),
            (g.dA, ref[2], 2 * c + n ** 0.5, 1, "dA"), (g.dD, ref[5], c + n ** 0.5, 0, "dD")):
        close(got, want, units, dims, what)


# ---------------------------------------------------------------- slow states

@pytest.mark.parametrize("b,d", SPLITS)
def test_scan_of_slow_states_errs_like_a_float32_loop(b, d):
    """Factors from 0.85 to 0.999 over 400 steps, where a one-sided error of the
    exponential would add up. The kernel makes the roundings of a plain float32
    loop and its exponentials' (2 units against 1): at most twice its distance
    from 64 bits in the root-mean-square sense."""
    n, N = 400, 16
    u, B, C, dout = rnd(1, b, n, d), rnd(2, b, n, N), rnd(3, b, n, N), rnd(4, b, n, d)
    delta = (rnd(5, b, n, d).abs() * 0.004 + 0.001).clamp(max=0.01)
    A = -torch.arange(1.0, N + 1, device="cuda").expand(d, N).contiguous()

    def loop(dtype):
        v = [t.to(dtype).requires_grad_(True) for t in (u, delta, A, B, C)]
        U, D, a, b_, c = v
        h, ys = torch.zeros(b, d, N, dtype=dtype, device="cuda"), []
        for t in range(n):
            h = torch.exp(D[:, t, :, None] * a) * h + (D[:, t] * U[:, t])[..., None] * b_[:, t, None]
            ys.append((h * c[:, t, None]).sum(-1))
        y = torch.stack(ys, 1)
        return [y.detach(), h.detach(), *torch.autograd.grad((y * dout.to(dtype)).sum(), v)]

    exact, plain = loop(torch.float64), loop(torch.float32)
    r = sq.selective_scan(u, delta, A, B, C, save_states=True)
    g = sq.selective_scan_backward(dout, u, delta, A, B, C, r.states)
    got = [r.out, r.final_state, g.du, g.ddelta, g.dA, g.dB, g.dC]
    off = lambda x, ref: ((x - ref).norm() / ref.norm()).item()
    for name, k, p, e in zip(("out", "final_state", "du", "ddelta", "dA", "dB", "dC"), got, plain, exact):
        assert off(k, e) <= 2 * off(p, e), (name, off(k, e), off(p, e))
    state = rnd(6, b, d, N)                          # one step at a time
    ref = [state.to(t).clone() for t in (torch.float64, F32)]
    for t in range(n):
        for h in ref:
            x = h.dtype
            h.mul_(torch.exp(delta[:, t, :, None].to(x) * A.to(x)))
            h.add_((delta[:, t].to(x) * u[:, t].to(x))[..., None] * B[:, t, None].to(x))
        sq.selective_scan_step(u[:, t], delta[:, t], A, B[:, t], C[:, t], state)
    assert off(state, ref[0]) <= 2 * off(ref[1], ref[0])


@pytest.mark.parametrize("b,d", SPLITS)
def test_scan_states_of_rate_zero_stay(b, d):
    """A = 0: the factor is 1 to the last bit, at every step and past the end, so
    a state without input keeps its bits."""
    n, N = 500, 16
    u, B = torch.zeros(b, n, d, device="cuda"), rnd(1, b, n, N)
    delta, A, h0 = rnd(2, b, n, d), full(0.0, d, N), rnd(3, b, d, N)
    for softplus in (True, False):
        r = sq.selective_scan(u, delta, A, B, B, delta_softplus=softplus, initial_state=h0,
                              save_states=True)
        assert torch.equal(r.final_state, h0)
        assert all(torch.equal(r.states[:, i], h0) for i in range(r.states.shape[1]))
    state = h0.clone()
    sq.selective_scan_step(u[:, 0], delta[:, 0], A, B[:, 0], B[:, 0], state, delta_softplus=True)
    assert torch.equal(state, h0)
    dfin = rnd(4, b, d, N)
    g = sq.selective_scan_backward(u, u, delta, A, B, B, r.states, dfinal_state=dfin)
    assert torch.equal(g.dinitial_state, dfin)


# ---------------------------------------------------------------- sizes

def test_lengths_that_wrap_around_are_refused():
    """Checked before any size is computed from them; nothing is launched."""
    h = capi.DeviceHandle(0)
    buf = torch.zeros(64, device="cuda").data_ptr()
    rows = capi.Rows(buf, 0, 0)
    conv = capi.ConvArgs(struct_size=ctypes.sizeof(capi.ConvArgs), taps=4, batch=1, channels=1,
                         length=2 ** 64 - 2, weight=buf, x=rows, y=rows)
    scan = capi.ScanArgs(struct_size=ctypes.sizeof(capi.ScanArgs), batch=1, channels=1, states=1,
                         groups=1, length=2 ** 64 - 1, u=rows, delta=rows, out=rows, B=rows, C=rows,
                         A=buf)
    for call, args in ((capi.lib().ferrum_causal_conv1d, conv), (capi.lib().ferrum_selective_scan, scan)):
        assert call(h.ptr, args, None) == capi.FERRUM_ERR_INVALID_ARG
        assert "too large" in capi.last_error()
    h.close()


# ---------------------------------------------------------------- streams and memory

def calls(seed=70):
    """Every operator that takes `out`: name, shape of out, call(out, stream)."""
    b, n, d, N = 4, 256, 512, 8
    x, z, w = rnd(seed, b, n, d), rnd(seed + 1, b, n, d), rnd(seed + 2, d, 4)
    A, bc = -rnd(seed + 3, d, N).abs(), rnd(seed + 4, b, n, N)
    cst, sst, nw = rnd(seed + 5, b, 3, d), rnd(seed + 6, b, d, N), rnd(seed + 7, d)
    xl, k = rnd(seed + 8, b, d, n), rnd(seed + 9, d, n, std=0.05)
    pos = torch.full((b,), n - 1, dtype=torch.int32, device="cuda")
    return [
        ("conv", (b, n, d), lambda o, s: sq.causal_conv1d(x, w, out=o, stream=s)),
        ("conv step", (b, d), lambda o, s: sq.causal_conv1d_step(x[:, 0], cst, w, out=o, stream=s)),
        ("scan", (b, n, d), lambda o, s: sq.selective_scan(x, z, A, bc, bc, delta_softplus=True,
                                                           out=o, stream=s).out),
        ("scan step", (b, d), lambda o, s: sq.selective_scan_step(
            x[:, 0], z[:, 0], A, bc[:, 0], bc[:, 0], sst, delta_softplus=True, out=o, stream=s)),
        ("norm after", (b, n, d), lambda o, s: sq.norm_after(x, nw, gate=z, out=o, stream=s)),
        ("long conv", (b, d, n), lambda o, s: sq.long_conv(xl, k, out=o, stream=s)),
        ("long step", (b, d), lambda o, s: sq.long_conv_step(xl[:, :, 0].contiguous(), xl, pos, k,
                                                             out=o, stream=s)),
    ]


@pytest.mark.parametrize("i", range(7))
def test_a_given_output_outlives_its_call_on_another_stream(i):
    """The caller drops `out` while the call still waits: its memory must not go
    to the next allocation of the caller's stream."""
    name, shape, call = calls()[i]
    s = torch.cuda.Stream()
    call(torch.empty(shape, device="cuda"), s)      # loads the kernels, which may wait
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.zeros(shape, device="cuda")
    out = torch.empty(shape, device="cuda")
    at = out.data_ptr()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(200_000_000)      # some 0.1 s in which the call waits
    call(out, s)
    del out
    assert not s.query(), "the call ran too early to tell"
    fresh = torch.zeros(shape, device="cuda")       # the same request as out's
    assert fresh.data_ptr() != at, name
    s.synchronize()
    assert not bool(fresh.any()), name


def test_outputs_that_share_memory_are_refused():
    b, n, d, N = 2, 40, 16, 4
    refused = pytest.raises(ValueError, match="share memory")
    buf, z, w = rnd(1, b, n + 1, d), rnd(2, b, n, d), rnd(3, d, 4)
    x, shifted = buf[:, 1:], buf[:, :-1]
    A, bc, nw = -rnd(4, d, N).abs(), rnd(5, b, n, N), rnd(6, d)
    keep = buf.clone()
    with refused:
        sq.causal_conv1d(x, w, out=shifted)
    with refused:
        sq.selective_scan(x, z, A, bc, bc, out=shifted)
    with refused:
        sq.selective_scan(z, z, A, x[..., :N], bc, out=x)            # B inside out
    with refused:
        sq.norm_after(z[0], nw, residual=x[0], out=shifted[0])
    line = rnd(7, b * d * (n + 8) + 1)
    with refused:
        sq.long_conv(line[1:1 + b * d * n].view(b, d, n), rnd(8, d, n), out=line[:b * d * n].view(b, d, n))
    st = rnd(9, 3 * b * 3 * d)
    old, nxt = st[:b * 3 * d].view(b, 3, d), st[d:d + b * 3 * d].view(b, 3, d)
    with refused:
        sq.causal_conv1d_step(z[:, 0], old, w, next_state=nxt)
    with refused:
        sq.causal_conv1d_step(z[:, 0], old, w, out=old[:, 0])
    with refused:
        sq.causal_conv1d_step(old[:, 1], old, w)                     # x inside the state
    st = rnd(10, 2 * b * d * N)
    old, nxt = st[:b * d * N].view(b, d, N), st[N:N + b * d * N].view(b, d, N)
    with refused:
        sq.selective_scan_step(z[:, 0], z[:, 1], A, bc[:, 0], bc[:, 0], old, next_state=nxt)
    with refused:
        sq.selective_scan_step(z[:, 0], z[:, 1], A, bc[:, 0], bc[:, 0], old,
                               out=st[:b * d].view(b, d))
    hist, pos = rnd(11, b, d, n), torch.zeros(b, dtype=torch.int32, device="cuda")
    with refused:
        sq.long_conv_step(z[:, 0], hist, pos, rnd(12, d, n), out=hist.view(-1)[:b * d].view(b, d))
    with pytest.raises(ValueError, match="overlap itself"):
        sq.long_conv_step(z[:, 0], hist[:1].expand(b, d, n), pos, rnd(12, d, n))
    assert torch.equal(buf, keep)


def test_outputs_beside_their_inputs_are_taken():
    """Columns of one array, and a state that is its own successor."""
    b, n, d = 2, 40, 16
    wide, w = rnd(1, b, n, 3 * d), rnd(2, d, 4)
    x = wide[..., d:2 * d]
    want = sq.causal_conv1d(x, w)
    sq.causal_conv1d(x, w, out=wide[..., 2 * d:])
    assert torch.equal(wide[..., 2 * d:], want)
    sq.norm_after(x, rnd(3, d), gate=wide[..., 2 * d:], out=wide[..., :d])
    st = rnd(4, b, 3, d)
    other = torch.empty_like(st)
    y = sq.causal_conv1d_step(x[:, 0], st, w, next_state=other)
    assert torch.equal(y, sq.causal_conv1d_step(x[:, 0], st, w, next_state=st))
    assert torch.equal(st, other)


class Exported:
    """An array of another library: only DLPack, and it notes the stream that its
    producer is asked to be ready for."""

    def __init__(self, t):
        self.t, self.asked = t, []

    def __dlpack_device__(self):
        return self.t.__dlpack_device__()

    def __dlpack__(self, *, stream=None, **kw):
        self.asked.append(stream)
        return self.t.__dlpack__(stream=stream, **kw)


def test_arrays_of_other_libraries():
    """Taken without a copy, ready for the stream that the call runs on."""
    b, n, d, N = 2, 40, 16, 4
    x, z, w, nw = rnd(1, b, n, d), rnd(2, b, n, d), rnd(3, d, 4), rnd(4, d)
    A, bc, k = -rnd(5, d, N).abs(), rnd(6, b, n, N), rnd(7, n, d)
    pos = torch.zeros(b, dtype=torch.int32, device="cuda")
    e = Exported
    for given, want in (
            (lambda **s: sq.causal_conv1d(e(x), e(w), e(nw), **s), sq.causal_conv1d(x, w, nw)),
            (lambda **s: sq.selective_scan(x, e(z), e(A), bc, e(bc), z=e(z), **s).out,
             sq.selective_scan(x, z, A, bc, bc, z=z).out),
            (lambda **s: sq.norm_before(e(x), nw, residual=e(z), **s)[0],
             sq.norm_before(x, nw, residual=z)[0]),
            (lambda **s: sq.norm_after(x, e(nw), gate=e(z), **s), sq.norm_after(x, nw, gate=z)),
            (lambda **s: sq.long_conv(e(x), k, **s), sq.long_conv(x, k)),
            (lambda **s: sq.causal_conv1d_step(e(x[:, 0]), e(z[:, :3].contiguous()), w, **s),
             sq.causal_conv1d_step(x[:, 0], z[:, :3].contiguous(), w))):
        assert torch.equal(given(), want)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        got = given(stream=s)
        s.synchronize()
        assert torch.equal(got, want)
    out = torch.empty_like(x)
    assert sq.causal_conv1d(e(x), w, out=e(out)).data_ptr() == out.data_ptr()
    s = torch.cuda.Stream()
    for stream, asked in ((None, 1), (s, s.cuda_stream), (s.cuda_stream, s.cuda_stream), (0, 1)):
        x2 = e(x)
        sq.causal_conv1d(x2, w, stream=stream)
        assert x2.asked == [asked]         # (1 is DLPack's number of the default stream)
    torch.cuda.synchronize()


def test_a_stream_of_a_wrong_type_is_refused():
    x, w = rnd(1, 4, 8), rnd(2, 8)
    for stream in ("s", -1, 1.5):
        with pytest.raises(ValueError, match="stream must be"):
            sq.norm_before(x, w, stream=stream)


def stream_calls():
    """Every operator, gradient and step: name, the input that changes, call(stream)."""
    b, n, d, N = 3, 70, 40, 8
    r = lambda i, *s, **k: rnd(200 + i, *s, **k)
    x, z, dy = r(0, b, n, d), r(1, b, n, d), r(2, b, n, d)
    w, nw, cs = r(3, d, 4), r(4, d), r(5, b, 3, d)
    A, B, C, h = -r(6, d, N).abs(), r(7, b, n, N), r(8, b, n, N), r(9, b, d, N)
    st = sq.selective_scan(x, z, A, B, C, delta_softplus=True, save_states=True).states
    flat, out2 = x.view(b * n, d), torch.empty_like(h)
    res = r(10, b * n, d)
    big, bk = r(11, 1, 2, 16385), r(12, 2, 16385, std=0.01)      # several passes
    few, fk, fdy = r(13, 9, 2, 300), r(14, 2, 300, std=0.05), r(15, 9, 2, 300)
    last = r(16, b, 300, d).transpose(1, 2)                      # channel-last
    lk, pos = r(17, d, 300, std=0.05), torch.full((b,), n - 1, dtype=torch.int32, device="cuda")
    hist, hk, x1, z1 = r(18, b, d, n), r(19, d, n), x[:, 0].contiguous(), z[:, 0].contiguous()
    nxt = torch.empty_like(cs)
    k = dict(delta_softplus=True)
    return [
        ("conv", x, lambda s: sq.causal_conv1d(x, w, initial_state=cs, return_final_state=True, stream=s)),
        ("conv gradient", dy, lambda s: sq.causal_conv1d_backward(dy, x, w, nw, stream=s)),
        ("conv step", x1, lambda s: (sq.causal_conv1d_step(x1, cs, w, next_state=nxt, stream=s), nxt)),
        ("scan", x, lambda s: sq.selective_scan(x, z, A, B, C, stream=s, save_states=True, **k)),
        ("scan gradient", dy, lambda s: sq.selective_scan_backward(dy, x, z, A, B, C, st, stream=s, **k)),
        ("scan step", x1, lambda s: (sq.selective_scan_step(
            x1, z1, A, B[:, 0], C[:, 0], h, next_state=out2, stream=s, **k), out2)),
        ("norm before", flat, lambda s: sq.norm_before(flat, nw, residual=res, scale=nw, stream=s)),
        ("norm before gradient", flat, lambda s: sq.norm_before_backward(
            res, flat, nw, nw, x=res, scale=nw, stream=s)),
        ("norm after", flat, lambda s: (sq.norm_after(flat, nw, gate=res, groups=2, stream=s),)),
        ("norm after gradient", flat, lambda s: sq.norm_after_backward(
            res, flat, nw, nw, gate=res, scale=nw, stream=s)),
        ("long conv, by definition", hist, lambda s: (sq.long_conv(hist[:, :, :50], hk[:, :50].contiguous(), nw, stream=s),)),
        ("long conv, channel-last", last, lambda s: (sq.long_conv(last, lk, nw, stream=s),)),
        ("long conv, several passes", big, lambda s: (sq.long_conv(big, bk, stream=s),)),
        ("long conv gradient", few, lambda s: sq.long_conv_backward(fdy, few, fk, stream=s)),
        ("long conv gradient, several passes", big, lambda s: sq.long_conv_backward(big, big, bk, stream=s)),
        ("long step", x1, lambda s: (sq.long_conv_step(x1, hist, pos, hk, stream=s),)),
    ]


@pytest.mark.parametrize("i", range(16))
def test_calls_run_on_the_given_stream(i):
    """An input changes on the stream, behind a delay; only a call on that same
    stream sees it, with all its passes and workspaces."""
    name, t, call = stream_calls()[i]
    old = [v.clone() for v in call(None) if v is not None]
    new = rnd(300, *t.shape)
    keep = t.clone()
    t.copy_(new)
    want = [v.clone() for v in call(None) if v is not None]
    assert not all(torch.equal(p, q) for p, q in zip(old, want))
    t.copy_(keep)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)           # some 10 ms
        t.copy_(new)
    got = call(s)
    s.synchronize()
    for p, q in zip((v for v in got if v is not None), want):
        assert torch.equal(p, q), name
