"""Gated recurrence, dropout and the loss on the GPU against plain
implementations in 64 bits.

Tolerances. An output is rounded once to its type: u(type) |ref| with u = 2^-24,
2^-11, 2^-8. What comes before runs in float32 and is bounded for each operator
where its test is, in units of 2^-24.
"""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from conftest import gpu_available

from ferrum_gpu import capi, sequence as sq

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# half the spacing of values below the normal range
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
TYPES = [torch.float32, torch.float16, torch.bfloat16]
F32, F64 = torch.float32, torch.float64
EPS = 2.0 ** -24


@pytest.fixture(autouse=True, scope="module")
def _gpu():
    if not gpu_available():
        pytest.skip("no B200")


def rnd(seed, *shape, dtype=F32, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to("cuda").to(dtype)


def within(got, ref, bound, what=""):
    """|got - ref| <= bound + its type's rounding, element by element."""
    assert tuple(got.shape) == tuple(ref.shape), what
    if ref.numel() == 0:
        return
    g, r = got.detach().double(), ref.detach().double()
    assert bool(torch.isfinite(g).all()), f"{what}: not finite"
    over = (g - r).abs() - (U[got.dtype] * r.abs() + TINY[got.dtype] + bound)
    assert over.max().item() <= 0, f"{what}: above its bound by {over.max().item():.3e}"


# ---------------------------------------------------------------- gated recurrence
# Units of 2^-24, relative: a sigmoid 6 (exponential 2 and its argument's rounding
# times |logit| < 6, sum, reciprocal), m = a - 1 the sigmoid's and 2, the root
# half of m's and 4, the input the root's, a sigmoid's and 2: below 20. A step
# changes the state by no more than twice its input, and adds m's error and one
# rounding, which live on for as many steps as the channel remembers, at most n: an
# error of (20 + 10 min(n, memory)) units of the largest state, memory being
# 1 / (1 - a) at the slowest gate. Gradients are sums of the same kind over the
# state's gradient: twice that; ddecay adds n steps of b sequences, each off by
# as much relative to its own size (and the sum's roundings, fewer).

def gates(x, ig, rg, decay):
    r, i = torch.sigmoid(rg), torch.sigmoid(ig)
    la = -decay * r
    return torch.exp(la), torch.sqrt(-torch.expm1(2 * la)) * i * x


def ref_recurrence(x, ig, rg, decay, h, lengths):
    b, n, d = x.shape
    a, u = gates(x, ig, rg, decay)
    h = torch.zeros(b, d, dtype=F64, device="cuda") if h is None else h
    out, zero = [], torch.zeros((), dtype=F64, device="cuda")
    for t in range(n):
        new = a[:, t] * h + u[:, t]
        if lengths is None:
            h = new
            out.append(h)
        else:
            on = (t < lengths.long())[:, None]
            h = torch.where(on, new, h)
            out.append(torch.where(on, h, zero))
    return (torch.stack(out, 1) if out else torch.zeros(b, 0, d, dtype=F64, device="cuda")), h


REC = [  # batch, length, channels, initial state, ragged
    (1, 1, 1, False, False),
    (2, 1, 33, True, False),
    (3, 7, 5, True, True),
    (2, 16, 64, True, False),
    (2, 17, 128, False, True),
    (4, 129, 96, True, True),
    (1, 300, 130, True, False),
    (5, 257, 1000, True, True),
    (2, 1030, 72, True, False),
    (1, 2500, 64, True, False),
    (3, 515, 513, False, True),
]


def rec_inputs(case, dtype, seed=0):
    b, n, d, state, ragged = case
    x, ig, rg, dout = (rnd(seed + k, b, n, d, dtype=dtype) for k in range(4))
    decay = torch.rand(d, generator=torch.Generator().manual_seed(seed + 5)).cuda() * 0.7 + 0.02
    h = rnd(seed + 6, b, d) if state else None
    ln = None
    if ragged:   # empty, full, half, beyond both ends of the range (clamped)
        ln = torch.tensor([(0, n, n // 2, n + 5, -3)[i % 5] for i in range(b)],
                          dtype=torch.int32, device="cuda")
        pad = torch.arange(n, device="cuda")[None] >= ln[:, None].long()
        for v in (x, ig, rg, dout):
            v[pad] = float("nan")         # never read
    return x, ig, rg, decay, h, ln, dout


def clean(v, ln):
    if ln is None:
        return v.double()
    pad = torch.arange(v.shape[1], device="cuda")[None] >= ln[:, None].long()
    return v.double().masked_fill(pad[..., None], 0.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", REC)
def test_recurrence(case, dtype):
    x, ig, rg, decay, h, ln, dout = rec_inputs(case, dtype)
    b, n, d = x.shape
    leaves = [clean(v, ln).requires_grad_() for v in (x, ig, rg)]
    leaves += [decay.double().requires_grad_(),
               (torch.zeros(b, d, device="cuda") if h is None else h).double().requires_grad_()]
    out_ref, fin_ref = ref_recurrence(*leaves, ln)
    r = sq.gated_recurrence(x, ig, rg, decay, initial_state=h, lengths=ln, save_states=True)
    c = (20 + 10 * min(n, 150)) * EPS       # sigmoid(-3) * 0.02 is the slowest step here
    top = max(out_ref.detach().abs().max().item(), leaves[4].detach().abs().max().item())
    within(r.out, out_ref, c * top, "out")
    within(r.final_state, fin_ref, c * top, "final state")
    assert tuple(r.states.shape) == (b, (n + 15) // 16, d)
    plain = sq.gated_recurrence(x, ig, rg, decay, initial_state=h, lengths=ln)
    assert plain.states is None and torch.equal(plain.out, r.out)
    dfin = rnd(77, b, d)
    loss = (out_ref * clean(dout, ln)).sum() + (fin_ref * dfin.double()).sum()
    want = torch.autograd.grad(loss, leaves)
    got = sq.gated_recurrence_backward(dout, x, ig, rg, decay, r.states, lengths=ln,
                                       dfinal_state=dfin)
    for g, w, what in zip(got, want, got._fields):
        scale = w.abs().max().item()
        if what == "ddecay":      # terms of the size of drg / (decay (1 - r)), all off alike
            per = want[2].abs() / (decay.double() * (1 - torch.sigmoid(leaves[2].detach())))
            scale = per.sum((0, 1))[None].clamp(min=top)
            assert ((g.double() - w).abs() <= 4 * c * scale[0] + U[F32] * w.abs()).all(), what
            continue
        within(g, w, 4 * c * max(scale, top), what)
    if ln is not None:
        pad = torch.arange(n, device="cuda")[None] >= ln[:, None].long()
        for v in (r.out, got.dx, got.dinput_gate, got.drecurrence_gate):
            assert not v[pad].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,d", [(1, 1), (3, 33), (7, 256), (256, 130)])
def test_recurrence_step(b, d, dtype):
    x, ig, rg = (rnd(k, b, d, dtype=dtype) for k in range(3))
    decay, h = rnd(4, d).abs(), rnd(5, b, d)
    a, u = gates(x.double(), ig.double(), rg.double(), decay.double())
    want = a * h.double() + u
    keep, nxt = h.clone(), torch.empty_like(h)
    y = sq.gated_recurrence_step(x, ig, rg, decay, h, next_state=nxt)
    assert torch.equal(h, keep)
    c = 30 * EPS * (h.double().abs() + x.double().abs())
    within(y, want, c, "out")
    within(nxt, want, c, "next state")
    y2 = sq.gated_recurrence_step(x, ig, rg, decay, h)
    assert torch.equal(y, y2) and torch.equal(h, nxt)


def test_recurrence_in_parts_and_steps():
    """A prompt in two calls and then token by token is the whole."""
    x, ig, rg, decay, h, _, _ = rec_inputs((2, 90, 40, True, False), F32)
    whole = sq.gated_recurrence(x, ig, rg, decay, initial_state=h)
    first = sq.gated_recurrence(x[:, :37], ig[:, :37], rg[:, :37], decay, initial_state=h)
    second = sq.gated_recurrence(x[:, 37:80], ig[:, 37:80], rg[:, 37:80], decay,
                                 initial_state=first.final_state)
    state, outs = second.final_state, [first.out, second.out]
    for t in range(80, 90):
        outs.append(sq.gated_recurrence_step(x[:, t], ig[:, t], rg[:, t], decay, state)[:, None])
    bound = 2 * (20 + 10 * 90) * EPS * whole.out.abs().max().item()
    within(torch.cat(outs, 1), whole.out.double(), bound)
    within(state, whole.final_state.double(), bound)


def test_recurrence_views():
    """Channels of wider rows, steps of a (length, batch) layout, own outputs."""
    b, n, d = 3, 70, 48
    wide = rnd(1, n, b, 3 * d + 5).transpose(0, 1)
    x, ig, rg = wide[..., 1:1 + d], wide[..., d + 1:2 * d + 1], wide[..., 2 * d + 3:3 * d + 3]
    decay = rnd(2, d).abs() * 0.3 + 0.01
    want = sq.gated_recurrence(x.contiguous(), ig.contiguous(), rg.contiguous(), decay)
    room = torch.full((b, n, 2 * d), 7.0, device="cuda")
    got = sq.gated_recurrence(x, ig, rg, decay, out=room[..., d:])
    bound = 2 * (20 + 10 * n) * EPS * want.out.abs().max().item()
    within(got.out, want.out.double(), bound)
    assert got.out.data_ptr() == room[..., d:].data_ptr() and bool((room[..., :d] == 7).all())


def test_recurrence_extremes():
    """Shut and open gates, a decay of 0 and one beyond the exponential's range."""
    n = 40
    x = rnd(1, 1, n, 8)
    ig = torch.zeros(1, n, 8, device="cuda")
    rg = torch.tensor([-float("inf"), -200.0, -95.0, 0.0, 95.0, 200.0, float("inf"), 0.0],
                      device="cuda").expand(1, n, 8).contiguous()
    decay = torch.tensor([1.0, 1.0, 1.0, 0.0, 200.0, 1.0, 1.0, 1e-30], device="cuda")
    h = rnd(2, 1, 8)
    r = sq.gated_recurrence(x, ig, rg, decay, initial_state=h, save_states=True)
    # never forgets and takes nothing in: the state stays, bit by bit
    for c in (0, 3):
        assert torch.equal(r.out[0, :, c], h[0, c].expand(n))
    # forgets everything at once: the root is 1, the output half the input
    within(r.out[0, :, 4], x[0, :, 4].double() / 2, 8 * EPS * x.abs().max().item())
    g = sq.gated_recurrence_backward(torch.ones_like(x), x, ig, rg, decay, r.states)
    for v in g:
        assert torch.isfinite(v).all()
    a, u = gates(x.double(), ig.double(), rg.double(), decay.double())
    want, _ = ref_recurrence(x.double(), ig.double(), rg.double(), decay.double(), h.double(), None)
    within(r.out, want, (20 + 10 * n) * EPS * want.abs().max().item())


def test_recurrence_long_memory_in_float32():
    """Factors up to 0.9999 over 4000 steps: errors do not add up in one
    direction. A float32 loop's own roundings, half a unit a step and random,
    make sqrt(4000) units of the largest state; four times that is allowed."""
    n, d = 4000, 64
    x, ig = rnd(1, 1, n, d), rnd(2, 1, n, d)
    rg = rnd(3, 1, n, d, std=0.1)
    decay = torch.logspace(-3.7, -0.5, d, device="cuda")
    want, fin = ref_recurrence(x.double(), ig.double(), rg.double(), decay.double(), None, None)
    got = sq.gated_recurrence(x, ig, rg, decay)
    err = (got.out.double() - want).abs().amax(1) / want.abs().amax(1)
    assert err.max().item() <= 4 * n ** 0.5 * EPS


def test_recurrence_empty():
    d = torch.ones(8, device="cuda")
    for b, n, c in ((2, 0, 8), (0, 5, 8), (2, 5, 0)):
        x = torch.zeros(b, n, c, device="cuda")
        h = rnd(1, b, c)
        r = sq.gated_recurrence(x, x, x, d[:c].contiguous(), initial_state=h, save_states=True)
        assert r.out.shape == x.shape and (b * c == 0 or n or torch.equal(r.final_state, h))
        g = sq.gated_recurrence_backward(x, x, x, x, d[:c].contiguous(), r.states, dfinal_state=h)
        assert g.dx.shape == x.shape and g.ddecay.shape == (c,)
        assert not g.ddecay.any() and (n or torch.equal(g.dinitial_state, h))


def test_recurrence_beyond_2_31_values():
    """The end of an array of more than 2^31 values, against a short call on that end:
    with memories of less than 40 steps (e^-0.45 a step and more), a start 400 steps
    earlier from zero leaves e^-180 of a difference."""
    n, d = 2 ** 21 + 100, 1040
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty(1, n, d, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    gate = torch.zeros(1, 1, 1, device="cuda", dtype=torch.bfloat16).expand(1, n, d).contiguous()
    decay = torch.full((d,), 0.9, device="cuda")
    whole = sq.gated_recurrence(x, gate, gate, decay, save_states=True)
    end = slice(n - 500, n)
    part = sq.gated_recurrence(x[:, end], gate[:, end], gate[:, end], decay)
    bound = 2 * (20 + 400) * EPS * 4.0
    within(whole.out[:, -100:], part.out[:, -100:].double(), 2.0 ** -8 * part.out[:, -100:].double().abs() + bound)
    within(whole.final_state, part.final_state.double(), bound)
    back = sq.gated_recurrence_backward(x, x, gate, gate, decay, whole.states)
    assert torch.isfinite(back.dx[:, -100:].float()).all() and bool(back.dx[:, -1].any())
    assert bool(back.dx[:, 0].any()) and torch.isfinite(back.ddecay).all()


# ---------------------------------------------------------------- dropout
# y = res + x * scale: the rounding of scale and of the product, then the sum's,
# which is the output's.

def philox(n, seed, offset=0):
    """Words of elements 0 .. n - 1, with Python's integers (Salmon et al. 2011)."""
    low, out = 0xFFFFFFFF, []
    for g in range((n + 3) // 4):
        c = [g & low, g >> 32, offset & low, (offset >> 32) & low]
        k = [seed & low, (seed >> 32) & low]
        for _ in range(10):
            p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & low, (p0 >> 32) ^ c[3] ^ k[1], p0 & low]
            k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
        out += c
    return torch.tensor(out[:n], device="cuda")


def test_philox_known_answers():
    """The published generator's vectors: counter and key all zeros, all ones."""
    assert [hex(v) for v in philox(4, 0).tolist()] == [
        "0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]


def drop_ref(x, p, keep, residual):
    y = torch.where(keep, x.double() / (1 - p) if p < 1 else torch.zeros_like(x.double()),
                    torch.zeros((), dtype=F64, device="cuda"))
    return y if residual is None else residual.double() + y


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("res", ["none", "same", "f32"])
@pytest.mark.parametrize("shape", [(1,), (7,), (2, 5), (3, 8), (129, 40), (2, 3, 33), (5, 1000)])
def test_dropout(shape, res, dtype):
    x = rnd(1, *shape, dtype=dtype)
    rt = {"none": dtype, "same": dtype, "f32": F32}[res]
    residual = None if res == "none" else rnd(2, *shape, dtype=rt)
    p, seed = 0.3, 0x123456789ABCDEF
    keep = (philox(x.numel(), seed, 5) >= int(p * 2 ** 32)).view(shape)
    y = sq.dropout(x, p, seed, offset=5, residual=residual)
    assert y.dtype == rt
    within(y, drop_ref(x, p, keep, residual), 2 * EPS * x.double().abs() / (1 - p))
    dy = rnd(3, *shape, dtype=rt)
    dx = sq.dropout_backward(dy, p, seed, offset=5, dtype=dtype)
    assert dx.dtype == dtype
    within(dx, drop_ref(dy, p, keep, None), 2 * EPS * dy.double().abs() / (1 - p))
    assert not dx[~keep].any()


def test_dropout_seeds_and_ends():
    x = rnd(1, 64, 256)
    t = torch.tensor([-3], device="cuda")
    same = [sq.dropout(x, 0.5, s) for s in (-3, 2 ** 64 - 3, t, t.view(()), np.int64(-3))]
    for y in same[1:]:
        assert torch.equal(y, same[0])
    for other in (sq.dropout(x, 0.5, 4), sq.dropout(x, 0.5, -3, offset=1),
                  sq.dropout(x, 0.5, -3, offset=-1), sq.dropout(x, 0.5, -3 + 2 ** 32)):
        # independent masks agree on half of 16384 values: 64 a standard deviation
        assert abs(((other != 0) == (same[0] != 0)).sum().item() - 8192) < 6 * 64
    assert torch.equal(sq.dropout(x, 0.0, 1), x)
    assert not sq.dropout(x, 1.0, 1).any()
    r = rnd(2, 64, 256)
    assert torch.equal(sq.dropout(x, 1.0, 1, residual=r), r)
    assert not sq.dropout_backward(x, 1.0, 1).any()
    big = rnd(3, 1024, 1024)
    for p in (0.1, 0.5, 0.9):
        kept = (sq.dropout(big, p, 9) != 0).sum().item()
        assert abs(kept - big.numel() * (1 - p)) < 6 * (big.numel() * p * (1 - p)) ** 0.5


def test_dropout_leaves_no_trace_of_dropped_values():
    x = torch.full((3, 257), float("nan"), device="cuda")
    keep = (philox(x.numel(), 11) >= int(0.4 * 2 ** 32)).view(3, 257)
    y = sq.dropout(x, 0.4, 11, residual=torch.ones_like(x))
    assert bool((y[~keep] == 1).all()) and bool(torch.isnan(y[keep]).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("channels,lead", [(40, 0), (40, 1), (33, 0), (64, 8), (1, 3)])
def test_dropout_strides_keep_the_mask(channels, lead, dtype):
    """The mask goes by an element's index, whatever its place in memory."""
    rows = 37
    wide = rnd(1, rows, channels + 24, dtype=dtype)
    x = wide[:, lead:lead + channels]
    room = torch.full((rows, channels + 16), 7.0, device="cuda", dtype=dtype)
    want = sq.dropout(x.contiguous(), 0.2, 5, residual=x.contiguous())
    got = sq.dropout(x, 0.2, 5, residual=wide[:, lead:lead + channels],
                     out=room[:, lead:lead + channels])
    assert torch.equal(got, want)
    assert bool((room[:, :lead] == 7).all()) and bool((room[:, lead + channels:] == 7).all())
    assert torch.equal(sq.dropout_backward(x, 0.2, 5), sq.dropout_backward(x.contiguous(), 0.2, 5))


def test_dropout_beyond_32_bits():
    """Elements beyond 2^32 have counters of their own."""
    n = (1 << 32) + 4096
    x = torch.ones(n, device="cuda", dtype=torch.bfloat16)
    y = sq.dropout(x, 0.5, 21)
    low = 0xFFFFFFFF
    for first in (0, (1 << 32) - 8, (1 << 32) + 4088):
        want = []
        for g in range(first // 4, first // 4 + 2):
            c, k = [g & low, g >> 32, 0, 0], [21, 0]
            for _ in range(10):
                p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
                c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & low, (p0 >> 32) ^ c[3] ^ k[1], p0 & low]
                k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
            want += [v >= 1 << 31 for v in c]
        assert (y[first:first + 8] != 0).tolist() == want


# ---------------------------------------------------------------- loss
# A logit is a sum of `width` exact products (16-bit types) or rounded ones, each
# of its additions off by at most 2 units of 2^-24 of the absolute sum (tensor
# cores cut off where others round): e = 2 (width + 1) 2^-24 (|x| |W|^T). A row's
# lse is off by its largest e and 8 units of its own size, 8 more for exponential
# and logarithm; the loss by the target's e besides. A softmax value p is off by
# p times (e + lse's error + 6 units), and rounded to the type of x before the
# gradients' products; those add 2 (vocab or tokens + pieces) units of the
# absolute sum.

def loss_case(tokens, width, vocab, dtype, masked, seed=0, scale=1.5):
    x = rnd(seed, tokens, width, dtype=dtype)
    w = rnd(seed + 1, vocab, width, dtype=dtype, std=scale / width ** 0.5)
    g = torch.Generator().manual_seed(seed + 2)
    t = torch.randint(vocab, (tokens,), generator=g)
    lost = torch.rand(tokens, generator=g) < masked
    t[lost] = torch.tensor([-100, vocab, -1, 2 ** 40])[torch.arange(int(lost.sum())) % 4]
    return x, w, t.cuda()


def loss_ref(x, w, t):
    xd, wd = x.double(), w.double()
    logits = xd @ wd.t()
    e = 2 * (x.shape[-1] + 1) * EPS * (xd.abs() @ wd.abs().t())
    lse = torch.logsumexp(logits, 1)
    ok = (t >= 0) & (t < w.shape[0])
    at = t.where(ok, torch.zeros_like(t))[:, None]
    loss = (lse - logits.gather(1, at)[:, 0]).where(ok, torch.zeros_like(lse))
    return logits, e, lse, ok, at, loss


def check_loss(x, w, t, dloss, dlse=None, r=None):
    logits, e, lse, ok, at, loss = loss_ref(x, w, t)
    off = e.amax(1) + 8 * EPS * (1 + lse.abs() + logits.abs().amax(1))
    r = sq.linear_cross_entropy(x, w, t) if r is None else r
    zero = torch.zeros_like(lse)
    within(r.lse, lse.where(ok, zero), off, "lse")
    within(r.loss, loss, 2 * off, "loss")
    assert not r.loss[~ok].any() and not r.lse[~ok].any()
    got = sq.linear_cross_entropy_backward(dloss, x, w, t, r.lse, dlse=dlse)
    one = dloss.double().where(ok, zero)[:, None]
    both = one + (0 if dlse is None else dlse.double().where(ok, zero)[:, None])
    p = torch.exp(logits - lse[:, None])
    hot = torch.zeros_like(p).scatter_(1, at, 1.0)
    grad = p * both - hot * one
    # rounded sums of two terms: each term's size counts
    u = U[x.dtype]
    size = p * both.abs() + hot * one.abs()
    err = p * both.abs() * (2 * off[:, None] + 6 * EPS) + 2 * EPS * size + u * grad.abs()
    err = err + 2.0 ** -126 * both.abs()      # exponentials below the normal range are 0
    if x.dtype == torch.float16:   # spacing of the scaled values near 0
        err = err + 2.0 ** -38 * (both.abs().max() + one.abs().max())
    xd, wd = x.double().masked_fill(~ok[:, None], 0.0), w.double()
    n, v = p.shape
    within(got.dx, grad @ wd, err @ wd.abs() + 2 * (v + 64) * EPS * (size @ wd.abs()), "dx")
    within(got.dweight, grad.t() @ xd, err.t() @ xd.abs() + 2 * (n + 64) * EPS * (size.t() @ xd.abs()),
           "dweight")
    assert not got.dx[~ok].any()
    return r, got


LOSS = [  # tokens, width, vocab, masked
    (1, 1, 1, 0.0),
    (1, 8, 2, 0.0),
    (3, 16, 5, 0.3),
    (8, 64, 1000, 0.0),
    (33, 72, 257, 0.3),
    (129, 100, 300, 0.3),
    (128, 128, 512, 0.0),
    (200, 333, 1001, 0.5),
    (257, 264, 1500, 1.0),
    (300, 512, 4099, 0.1),
    (700, 200, 9000, 0.1),
    (5, 2048, 3001, 0.2),
    (70, 24, 3, 0.2),
    (100, 320, 5000, 0.1),
    (64, 136, 20011, 0.1),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", LOSS)
def test_loss(case, dtype):
    tokens, width, vocab, masked = case
    x, w, t = loss_case(tokens, width, vocab, dtype, masked)
    check_loss(x, w, t, rnd(9, tokens).abs() + 0.1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,width,vocab", [(40000, 16, 9000), (256, 64, 700000), (65, 40, 70000)])
def test_loss_in_pieces_of_the_vocabulary(tokens, width, vocab, dtype):
    """Many tokens in three pieces; many words in two, with dx in slabs besides."""
    x, w, t = loss_case(tokens, width, vocab, dtype, 0.1)
    d = torch.full((tokens,), 1.0 if dtype == torch.float16 else 1.0 / tokens, device="cuda")
    check_loss(x, w, t, d)


@pytest.mark.parametrize("dtype", TYPES)
def test_loss_normaliser_gradient(dtype):
    x, w, t = loss_case(150, 96, 700, dtype, 0.2)
    check_loss(x, w, t, rnd(9, 150), rnd(10, 150, std=0.1))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [2.0 ** -30, 2.0 ** 20])
def test_loss_gradients_of_any_size(scale, dtype):
    """Tiny gradients (a mean over many tokens) keep their relative accuracy in
    between; their outputs are float32's range or the type's."""
    x, w, t = loss_case(140, 64, 600, dtype, 0.1)
    d = (rnd(9, 140).abs() + 0.1) * scale
    if dtype == torch.float16:
        d = d.clamp(2.0 ** -10, 16.0)       # its outputs' own range
    check_loss(x, w, t, d)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("count", [1, 777, 1000])
def test_loss_gradients_do_not_share_an_error(count, dtype):
    """A mean over tokens: every target's value is nearly -1 / count, and a rounding
    that all had alike would be a relative error of the whole, up to u. Rounding the
    outputs alone leaves u sqrt(E[1 / m^2] / 3) = 0.425 u over mantissas m in [1, 2);
    the softmax's part, below 0.2 of the whole here, adds as much of its own size:
    0.425 u sqrt(1 + 0.2^2) < 0.5 u."""
    x, w, t = loss_case(count, 256, 3000, dtype, 0.0)
    scale = 1024.0 if dtype == torch.float16 else 1.0
    d = torch.full((count,), scale / count, device="cuda")
    r = sq.linear_cross_entropy(x, w, t)
    g = sq.linear_cross_entropy_backward(d, x, w, t, r.lse)
    p = torch.softmax(x.double() @ w.double().t(), 1)
    p[torch.arange(count, device="cuda"), t] -= 1
    p *= scale / count
    for got, ref in ((g.dx, p @ w.double()), (g.dweight, p.t() @ x.double())):
        assert ((got.double() - ref).norm() / ref.norm()).item() <= 0.5 * U[dtype]


def test_loss_rows_without_a_target_are_not_read():
    for dtype in TYPES:
        x, w, t = loss_case(140, 64, 600, dtype, 0.4)
        bad = (t < 0) | (t >= 600)
        d, e = rnd(9, 140).abs(), rnd(10, 140)
        want = sq.linear_cross_entropy(x, w, t)
        ref = sq.linear_cross_entropy_backward(d, x, w, t, want.lse, dlse=e)
        x2, d2, e2 = x.clone(), d.clone(), e.clone()
        x2[bad], d2[bad], e2[bad] = float("nan"), float("inf"), float("nan")
        lse2 = want.lse.clone()
        lse2[bad] = float("nan")
        got = sq.linear_cross_entropy(x2, w, t)
        assert torch.equal(got.loss, want.loss) and torch.equal(got.lse, want.lse)
        g = sq.linear_cross_entropy_backward(d2, x2, w, t, lse2, dlse=e2)
        assert torch.equal(g.dx, ref.dx) and torch.equal(g.dweight, ref.dweight)


@pytest.mark.parametrize("dtype", TYPES)
def test_loss_extreme_logits(dtype):
    """Logits far apart: one takes all of the softmax, the others vanish."""
    x, w, t = loss_case(70, 64, 500, dtype, 0.0, scale=60.0)
    check_loss(x, w, t, torch.ones(70, device="cuda"))
    # infinite logits, of either sign
    for tokens in (3, 70):
        x = torch.ones(tokens, 8, device="cuda", dtype=dtype)
        w = torch.zeros(300, 8, device="cuda", dtype=dtype)
        w[7, 0] = float("-inf")
        t = torch.tensor([0, 299, 7], device="cuda").repeat(24)[:tokens].contiguous()
        r = sq.linear_cross_entropy(x, w, t)
        want = torch.tensor([299.0]).log().item()
        assert torch.allclose(r.lse, torch.full_like(r.lse, want), rtol=1e-6, atol=0)
        assert r.loss[2].item() == float("inf")
        w[9, 0] = float("inf")
        r = sq.linear_cross_entropy(x, w, t)
        assert bool(torch.isinf(r.lse).all())
        x[1, 3] = float("nan")
        w[7, 0] = w[9, 0] = 0.0
        r = sq.linear_cross_entropy(x, w, t)      # a row keeps its NaN to itself
        assert torch.isnan(r.loss).tolist() == [i == 1 for i in range(tokens)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lead,pad", [(0, 8), (8, 8), (1, 3), (3, 2)])
def test_loss_views(lead, pad, dtype):
    """Rows inside wider ones, at starts and strides that 16 bytes do not divide."""
    tokens, width, vocab = 90, 96, 333
    xw, ww, t = loss_case(tokens, width + lead + pad, vocab, dtype, 0.1)
    x, w = xw[:, lead:lead + width], ww[:, lead:lead + width]
    check_loss(x, w, t, torch.ones(tokens, device="cuda"))


def test_loss_shapes_and_empty():
    x, w, t = loss_case(24, 40, 77, F32, 0.0)
    flat = sq.linear_cross_entropy(x, w, t)
    cube = sq.linear_cross_entropy(x.view(2, 3, 4, 40), w, t.view(2, 3, 4))
    assert torch.equal(cube.loss, flat.loss.view(2, 3, 4))
    one = sq.linear_cross_entropy(x[0], w, t[0])
    assert one.loss.shape == () and torch.equal(one.loss, sq.linear_cross_entropy(x[:1], w, t[:1]).loss[0])
    for dtype in TYPES:
        e = sq.linear_cross_entropy(x[:0].to(dtype), w.to(dtype), t[:0])
        assert e.loss.shape == (0,)
        g = sq.linear_cross_entropy_backward(e.loss, x[:0].to(dtype), w.to(dtype), t[:0], e.lse)
        assert g.dx.shape == (0, 40) and not g.dweight.any()


def test_loss_against_differences():
    x, w, t = loss_case(6, 12, 50, F32, 0.2)
    d = torch.ones(6, device="cuda")
    r = sq.linear_cross_entropy(x, w, t)
    g = sq.linear_cross_entropy_backward(d, x, w, t, r.lse)
    step = 2.0 ** -7
    for i, j in ((0, 0), (2, 5), (5, 11)):
        for leaf, grad in ((x, g.dx), (w, g.dweight)):
            up, down = leaf.clone(), leaf.clone()
            up[i, j] += step
            down[i, j] -= step
            run = lambda v: sq.linear_cross_entropy(*((v, w) if leaf is x else (x, v)), t).loss.double().sum()
            slope = ((run(up) - run(down)) / (2 * step)).item()
            # third derivatives below 1 x step^2 / 6, the losses' rounding over the step
            assert abs(slope - grad[i, j].item()) < 6 * step ** 2 + 6 * 64 * EPS / step


# ---------------------------------------------------------------- all of them
# Streams, captured graphs, repetition, refusals.

def calls(dtype=torch.bfloat16):
    """Each operator as a call on fixed inputs that returns its outputs."""
    x, ig, rg, decay, h, ln, dout = rec_inputs((3, 300, 200, True, True), dtype)
    lx, lw, lt = loss_case(200, 128, 1500, dtype, 0.2)
    dl = torch.ones(200, device="cuda")
    states = sq.gated_recurrence(x, ig, rg, decay, initial_state=h, lengths=ln, save_states=True).states
    lse = sq.linear_cross_entropy(lx, lw, lt).lse
    seed = torch.tensor([77], device="cuda")
    step = [v[:, 0].nan_to_num().contiguous() for v in (x, ig, rg)]
    nxt = torch.empty_like(h)
    return {
        "recurrence": lambda **k: sq.gated_recurrence(x, ig, rg, decay, initial_state=h, lengths=ln,
                                                      save_states=True, **k),
        "recurrence_backward": lambda **k: sq.gated_recurrence_backward(
            dout, x, ig, rg, decay, states, lengths=ln, dfinal_state=h, **k),
        "recurrence_step": lambda **k: (sq.gated_recurrence_step(*step, decay, h, next_state=nxt, **k), nxt),
        "dropout": lambda **k: (sq.dropout(lx, 0.3, seed, residual=lx.float(), **k),),
        "dropout_backward": lambda **k: (sq.dropout_backward(lx, 0.3, seed, **k),),
        "loss": lambda **k: sq.linear_cross_entropy(lx, lw, lt, **k),
        "loss_backward": lambda **k: sq.linear_cross_entropy_backward(dl, lx, lw, lt, lse, **k),
    }


NAMES = ["recurrence", "recurrence_backward", "recurrence_step", "dropout", "dropout_backward",
         "loss", "loss_backward"]


def same(a, b):
    assert len(a) == len(b)
    for u, v in zip(a, b):
        assert (u is None and v is None) or torch.equal(u.nan_to_num(), v.nan_to_num())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", NAMES)
def test_results_repeat(name, dtype):
    call = calls(dtype)[name]
    first = [None if v is None else v.clone() for v in call()]
    for _ in range(4):
        same(call(), first)


@pytest.mark.parametrize("name", NAMES)
def test_other_stream(name):
    call = calls()[name]
    want = [None if v is None else v.clone() for v in call()]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    got = call(stream=s)
    s.synchronize()
    same(got, want)
    got = call(stream=s.cuda_stream)
    s.synchronize()
    same(got, want)


@pytest.mark.parametrize("dtype", [F32, torch.bfloat16])
@pytest.mark.parametrize("name", NAMES)
def test_captured_twice_and_replayed_at_once(name, dtype):
    """Two graphs of the same call, replayed side by side on two streams."""
    call = calls(dtype)[name]
    want = [None if v is None else v.clone() for v in call()]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2 if name != "recurrence_step" else 1):   # (a step's state is one array)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call())
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o in outs:
        same(o, want)


def test_a_captured_dropout_draws_by_the_seed_in_memory():
    x = rnd(1, 64, 64)
    seed = torch.tensor([1], device="cuda")
    sq.dropout(x, 0.5, seed)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = sq.dropout(x, 0.5, seed)
    for s in (1, 5, 1):
        seed.fill_(s)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, sq.dropout(x, 0.5, s))


def test_together_as_a_training_step():
    """Mixer, dropout onto the residual and loss with all their gradients, against
    the same in 64 bits."""
    b, n, d, v, p = 2, 50, 32, 300, 0.25
    x, ig, rg, decay, h, _, _ = rec_inputs((b, n, d, True, False), F32)
    w, t = rnd(20, v, d, std=d ** -0.5), torch.randint(v, (b, n), device="cuda")
    res = rnd(21, b, n, d)
    r = sq.gated_recurrence(x, ig, rg, decay, initial_state=h, save_states=True)
    y = sq.dropout(r.out, p, 3, residual=res)
    ce = sq.linear_cross_entropy(y, w, t)
    dl = torch.full((b, n), 1.0 / (b * n), device="cuda")
    gl = sq.linear_cross_entropy_backward(dl, y, w, t, ce.lse)
    gd = sq.dropout_backward(gl.dx, p, 3)
    gr = sq.gated_recurrence_backward(gd, x, ig, rg, decay, r.states)
    leaves = [q.double().requires_grad_() for q in (x, ig, rg, decay, h, w, res)]
    out, _ = ref_recurrence(*leaves[:5], None)
    keep = (philox(b * n * d, 3) >= int(p * 2 ** 32)).view(b, n, d)
    yy = leaves[6] + torch.where(keep, out / (1 - p), torch.zeros((), dtype=F64, device="cuda"))
    loss = torch.nn.functional.cross_entropy((yy @ leaves[5].t()).view(-1, v), t.view(-1))
    want = torch.autograd.grad(loss, leaves)
    # each value passes the recurrence's bound (n steps), the loss's products, and back
    c = 8 * (20 + 10 * n + 2 * (d + v)) * EPS
    assert abs(ce.loss.double().mean().item() - loss.item()) <= c * loss.item()
    for g, q in zip((gr.dx, gr.dinput_gate, gr.drecurrence_gate, gr.ddecay, gr.dinitial_state,
                     gl.dweight, gl.dx), want):
        assert (g.double() - q).abs().max().item() <= c * q.abs().max().item()


def test_refusals():
    x, g2 = rnd(1, 2, 3, 8), rnd(2, 2, 8)
    d = rnd(3, 8).abs()
    w, t = rnd(4, 20, 8), torch.zeros(2, 3, dtype=torch.int64, device="cuda")
    f = torch.zeros(2, 3, device="cuda")
    bad = {
        "input_gate must be float32": lambda: sq.gated_recurrence(x, x.half(), x, d),
        "recurrence_gate must have shape": lambda: sq.gated_recurrence(x, x, x[:, :2], d),
        "decay must have shape": lambda: sq.gated_recurrence(x, x, x, d[:4]),
        "decay is required": lambda: sq.gated_recurrence(x, x, x, None),
        "decay must be float32": lambda: sq.gated_recurrence(x, x, x, d.half()),
        "lengths must be int32": lambda: sq.gated_recurrence(x, x, x, d, lengths=t[:, 0].contiguous()),
        "initial_state must have shape": lambda: sq.gated_recurrence(x, x, x, d, initial_state=d),
        "x must have 3 dimensions": lambda: sq.gated_recurrence(g2, g2, g2, d),
        "out must not share memory": lambda: sq.gated_recurrence(x, x, x, d, out=x),
        "states must have shape": lambda: sq.gated_recurrence_backward(x, x, x, x, d, g2),
        "states is required": lambda: sq.gated_recurrence_backward(x, x, x, x, d, None),
        "dout must have shape": lambda: sq.gated_recurrence_backward(x[:1], x, x, x, d, g2[:, None]),
        "state must have shape": lambda: sq.gated_recurrence_step(g2, g2, g2, d, d),
        "state is required": lambda: sq.gated_recurrence_step(g2, g2, g2, d, None),
        "state must not share": lambda: sq.gated_recurrence_step(g2, g2, g2, d, g2),
        r"p must be in \[0, 1\]": lambda: sq.dropout(x, 1.5, 1),
        "p must be in .*nan": lambda: sq.dropout(x, float("nan"), 1),
        "seed must be an integer": lambda: sq.dropout(x, 0.5, 1.5),
        "seed must be int64": lambda: sq.dropout(x, 0.5, d[:1]),
        "seed must be an integer or a tensor of one": lambda: sq.dropout(x, 0.5, t[0]),
        "seed must be a CUDA tensor": lambda: sq.dropout(x, 0.5, torch.tensor([1])),
        "residual must be float32": lambda: sq.dropout(x, 0.5, 1, residual=x.half()),
        "residual must have shape": lambda: sq.dropout(x, 0.5, 1, residual=x[:1]),
        "out must be float32": lambda: sq.dropout(x, 0.5, 1, out=x.half()),
        "out must not share": lambda: sq.dropout(x, 0.5, 1, residual=x.clone(), out=x),
        "dtype must be float32, float16": lambda: sq.dropout_backward(x, 0.5, 1, dtype=torch.float64),
        "dtype must be float16 ": lambda: sq.dropout_backward(x.half(), 0.5, 1, dtype=F32),
        "weight must be .vocabulary": lambda: sq.linear_cross_entropy(x, w[:, :4], t),
        "weight must be float32": lambda: sq.linear_cross_entropy(x, w.half(), t),
        "targets must be int64": lambda: sq.linear_cross_entropy(x, w, t.int()),
        "targets must have shape": lambda: sq.linear_cross_entropy(x, w, t[0]),
        "lse must be float32": lambda: sq.linear_cross_entropy_backward(f, x, w, t, f.half()),
        "lse is required": lambda: sq.linear_cross_entropy_backward(f, x, w, t, None),
        "dloss must have shape": lambda: sq.linear_cross_entropy_backward(f[0], x, w, t, f),
        "dloss must be contiguous": lambda: sq.linear_cross_entropy_backward(
            f[:1, :1].expand(2, 3), x, w, t, f),
        "collapse to one stride": lambda: sq.linear_cross_entropy(
            x.transpose(0, 1), w, t.t().contiguous()),
    }
    for match, call in bad.items():
        with pytest.raises(ValueError, match=match):
            call()


def test_c_refusals():
    """What the torch calls cannot send: each is refused before any launch."""
    dev = capi.DeviceHandle(0)
    lib = capi.lib()

    def refused(name, match, **fields):
        block = capi.SEQ_SIGNATURES[name]
        args = block(struct_size=ctypes.sizeof(block), **fields)
        assert getattr(lib, name)(dev.ptr, ctypes.byref(args), None) == capi.FERRUM_ERR_INVALID_ARG
        assert match in capi.last_error()

    big, p = 1 << 62, 4096
    refused("ferrum_gated_recurrence", "dtype", dtype=9)
    refused("ferrum_gated_recurrence", "too large", batch=big, length=big, channels=big)
    refused("ferrum_gated_recurrence", "too large", batch=0, length=(1 << 64) - 1, channels=1)
    refused("ferrum_gated_recurrence", "decay is NULL", batch=1, length=1, channels=1)
    refused("ferrum_gated_recurrence_step", "length must be 1", batch=0, length=2, channels=1, decay=p)
    refused("ferrum_dropout", "p must be", p=2.0)
    refused("ferrum_dropout", "residual_dtype", dtype=1, residual_dtype=2)
    refused("ferrum_dropout", "too large", rows=big, channels=big)
    refused("ferrum_dropout", "x is NULL", rows=1, channels=1)
    refused("ferrum_linear_cross_entropy", "width", tokens=1, vocab=1)
    refused("ferrum_linear_cross_entropy", "vocab", tokens=1, width=1)
    refused("ferrum_linear_cross_entropy", "below 2^31", tokens=big, width=1, vocab=1)
    refused("ferrum_linear_cross_entropy", "x is NULL", tokens=1, width=1, vocab=1)
    refused("ferrum_linear_cross_entropy_bwd", "dweight is NULL", tokens=0, width=1, vocab=1, weight=p)
