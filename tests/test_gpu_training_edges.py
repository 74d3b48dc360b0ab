"""Recurrence, dropout and the loss at their edges: clusters of blocks, decays on
both sides of the short form, infinities, sizes near a limit.

Tolerances as in test_gpu_training_ops.py, whose helpers these tests use: an
output's own rounding, and a bound in units of 2^-24 that is derived beside each
test.
"""

from __future__ import annotations

import ctypes
import threading

import pytest
import torch

from conftest import gpu_available
from test_gpu_training_ops import EPS, F32, TYPES, U, clean, loss_case, ref_recurrence, rnd, within
from test_training_edges import words

from ferrum_gpu import capi, sequence as sq

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def _gpu():
    if not gpu_available():
        pytest.skip("no B200")


# ---------------------------------------------------------------- clusters

# Batches that make clusters of 8, 4, 2 and 1 blocks: 32 or 64 channels a block, twice
# the blocks as long as there are no more than 296.
BATCHES = [3, 7, 15, 30, 60]


def lengths_of(b, n, kind):
    if kind == "empty":
        ln = [0] * b
    elif kind == "one":          # a single sequence has steps
        ln = [n if i == b // 2 else 0 for i in range(b)]
    else:
        ln = [(0, n, 1, n // 2, 0, n - 1, 17)[i % 7] for i in range(b)]
    return torch.tensor(ln, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["empty", "one", "mixed"])
@pytest.mark.parametrize("b", BATCHES)
def test_clusters_with_empty_sequences(b, kind, dtype):
    """Blocks without a step hand on their state at once, before others of their cluster
    have read anything: states pass through bit by bit, again and again the same."""
    n, d = 700, 200
    x, ig, rg, dout = (rnd(k, b, n, d, dtype=dtype) for k in range(4))
    ln = lengths_of(b, n, kind)
    none = (ln == 0).cpu()
    decay, h, dfin = rnd(5, d).abs() * 0.3 + 0.01, rnd(6, b, d), rnd(7, b, d)
    first = None
    for _ in range(20):
        r = sq.gated_recurrence(x, ig, rg, decay, initial_state=h, lengths=ln, save_states=True)
        g = sq.gated_recurrence_backward(dout, x, ig, rg, decay, r.states, lengths=ln,
                                         dfinal_state=dfin)
        # (saved states behind a sequence's end are those at its end)
        got = [r.out, r.final_state, r.states, *g]
        first = got if first is None else first
        for u, v in zip(got, first):
            assert torch.equal(u, v)
    assert torch.equal(first[1][none], h[none])
    assert torch.equal(g.dinitial_state[none], dfin[none])
    for v in (r.out, g.dx, g.dinput_gate, g.drecurrence_gate):
        assert not v[none].any()


# ---------------------------------------------------------------- decays

def decays(kind, d):
    """`mild` channels take the recurrence's short form, `strong` ones the general one, a
    warp with both of them the general one for all; log-uniform up to 20."""
    u = torch.rand(d, generator=torch.Generator().manual_seed(d)).cuda()
    mild, strong = 0.01 * 100 ** u, 1.001 * 20 ** u
    if kind == "mild":
        return mild
    if kind == "strong":
        return strong
    if kind == "groups":         # 64 channels of one kind, then 64 of the other
        return torch.where(torch.arange(d, device="cuda") // 64 % 2 == 0, mild, strong)
    return torch.where(torch.arange(d, device="cuda") % 5 == 3, strong, mild)


def check_recurrence(x, ig, rg, decay, h, ln, dout, dfin, memory):
    """All outputs and gradients against 64 bits. A step adds 10 units of 2^-24 and its
    input 20, which live on for `memory` steps; gradients are sums of the same kind
    over the state's gradient: four times that (test_gpu_training_ops.py has the
    derivation). drg is ddecay's term times decay (1 - r), ddecay the sum of its terms."""
    b, n, d = x.shape
    leaves = [clean(v, ln).requires_grad_() for v in (x, ig, rg)]
    leaves += [decay.double().requires_grad_(), h.double().requires_grad_()]
    out_ref, fin_ref = ref_recurrence(*leaves, ln)
    want = torch.autograd.grad((out_ref * clean(dout, ln)).sum() + (fin_ref * dfin.double()).sum(), leaves)
    r = sq.gated_recurrence(x, ig, rg, decay, initial_state=h, lengths=ln, save_states=True)
    got = sq.gated_recurrence_backward(dout, x, ig, rg, decay, r.states, lengths=ln, dfinal_state=dfin)
    c = (20 + 10 * min(n, memory)) * EPS
    top = max(out_ref.detach().abs().max().item(), h.abs().max().item())
    within(r.out, out_ref, c * top, "out")
    within(r.final_state, fin_ref, c * top, "final state")
    for g, w, what in zip(got, want, got._fields):
        if what == "ddecay":
            per = want[2].abs() / (decay.double() * (1 - torch.sigmoid(leaves[2].detach())))
            assert ((g.double() - w).abs() <= 4 * c * per.sum((0, 1)).clamp(min=top) + U[F32] * w.abs()).all(), what
        else:
            within(g, w, 4 * c * max(w.abs().max().item(), top), what)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("kind", ["mild", "strong", "groups", "mixed"])
@pytest.mark.parametrize("b,n,d", [(3, 1300, 200), (7, 700, 198), (15, 300, 200), (60, 200, 130), (2, 40, 77)])
def test_recurrence_decays(b, n, d, kind, ragged, dtype):
    """Full warps of the short and the general form, over several turns, in clusters of
    8, 4, 2 and 1 blocks, whole and ragged."""
    x, ig, rg, dout = (rnd(k, b, n, d, dtype=dtype) for k in range(4))
    ln = lengths_of(b, n, "mixed") if ragged else None
    if ragged:
        pad = torch.arange(n, device="cuda")[None] >= ln[:, None].long()
        for v in (x, ig, rg, dout):
            v[pad] = float("nan")
    # decays from 0.01 on, at gates whose mean over 200 steps is above 0.45
    check_recurrence(x, ig, rg, decays(kind, d), rnd(6, b, d), ln, dout, rnd(7, b, d), 222)


def test_recurrence_extreme_gates_have_gradients():
    """Shut and open gates and a decay that forgets at once: where the root is not 0 the
    gradients are the formula's, where it is 0 (a = 1) the gradient through it is 0."""
    n = 40
    x, dout = rnd(1, 1, n, 6), rnd(3, 1, n, 6)
    ig = torch.zeros(1, n, 6, device="cuda")
    rg = torch.tensor([-20.0, 0.0, 20.0, 0.0, -200.0, 0.0], device="cuda").expand(1, n, 6).contiguous()
    decay = torch.tensor([1.0, 200.0, 1.0, 80.0, 1.0, 0.0], device="cuda")
    h = rnd(2, 1, 6)
    r = sq.gated_recurrence(x, ig, rg, decay, initial_state=h, save_states=True)
    g = sq.gated_recurrence_backward(dout, x, ig, rg, decay, r.states)
    wide = [v[..., :4].double().requires_grad_() for v in (x, ig, rg, decay, h)]
    out, _ = ref_recurrence(*wide, None)
    want = torch.autograd.grad((out * dout[..., :4].double()).sum(), wide)
    # sigmoid(-20)'s exponential: its argument's rounding is 20 units more; the root of
    # its 1 - a^2 divides what the state's gradients, sums of n terms, are off by
    c = 4 * (20 + 20 + 10 * n) * EPS
    for v, w, what in zip(g, want, g._fields):
        err, size = (v[..., :4].double() - w).abs(), w.abs()
        assert (err.flatten(0, -2).amax(0) <= c * size.flatten(0, -2).amax(0).clamp(min=1e-30)).all() \
            if what != "ddecay" else (err <= c * size + c).all(), what
    # a = 1: nothing goes in, the state's gradient passes on as it is
    back = dout[0, :, 4:].double().flip(0).cumsum(0).flip(0)
    assert not g.dx[..., 4:].any() and not g.dinput_gate[..., 4:].any() and not g.drecurrence_gate[..., 4:].any()
    within(g.dinitial_state[:, 4:], back[:1], n * EPS * dout.double().abs().sum(1)[:, 4:])
    # ddecay = -sum r h G: r is 0, or 1/2 of a state that stands still
    assert g.ddecay[4].item() == 0
    term = back[:, 1] * h[0, 5].double() / 2
    assert abs(g.ddecay[5].item() + term.sum().item()) <= 2 * n * EPS * term.abs().sum().item()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,n,d", [(2, 1, 8), (3, 1300, 96), (7, 300, 130), (80, 90, 64)])
def test_a_recurrence_keeps_infinities(b, n, d, dtype):
    """a > 0, so an infinite state stays infinite, whatever the factors and however they
    are joined; only infinities of both signs make NaN. Other channels do not see it."""
    x, ig, rg = (rnd(k, b, n, d, dtype=dtype) for k in range(3))
    decay, h = decays("mixed", d), rnd(6, b, d)
    ln = lengths_of(b, n, "mixed")
    plain = sq.gated_recurrence(x, ig, rg, decay, initial_state=h, lengths=ln, save_states=True)
    inf, t = float("inf"), n // 3
    x2, h2 = x.clone(), h.clone()
    h2[:, 0], h2[:, 3], h2[:, 6] = inf, -inf, inf
    x2[:, t, 1], x2[:, t, 2] = inf, -inf
    x2[:, n // 2, 6] = -inf
    r = sq.gated_recurrence(x2, ig, rg, decay, initial_state=h2, lengths=ln, save_states=True)
    out, fin = ref_recurrence(*(v.double() for v in (x2, ig, rg, decay, h2)), ln)
    hit = [0, 1, 2, 3, 6]
    rest = [c for c in range(d) if c not in hit]
    for got, want in ((r.out, out), (r.final_state, fin)):
        off = ~torch.isfinite(want)
        assert torch.equal(got[off].double().nan_to_num(7.0, 8.0, 9.0), want[off].nan_to_num(7.0, 8.0, 9.0))
        top = h.abs().max().clamp(min=out[~torch.isinf(out)].nan_to_num().abs().max()).item()
        within(got[~off], want[~off], (20 + 10 * min(n, 222)) * EPS * top)
    for u, v in ((r.out, plain.out), (r.final_state, plain.final_state), (r.states, plain.states)):
        assert torch.equal(u[..., rest], v[..., rest])
    # token by token
    step = [v[:, 0].contiguous() for v in (x2, ig, rg)]
    want, _ = ref_recurrence(*(v[:, None].double() for v in step), decay.double(), h2.double(), None)
    y = sq.gated_recurrence_step(*step, decay, h2)
    for got in (y, h2):
        assert torch.equal(torch.isfinite(got), torch.isfinite(want[:, 0]))
        off = torch.isinf(want[:, 0])
        assert torch.equal(got[off].double(), want[:, 0][off])


@pytest.mark.parametrize("dtype", TYPES)
def test_a_gradient_behind_the_end_passes_on_as_it_is(dtype):
    """The final state's gradient is the initial one's where a sequence has no step."""
    b, n, d = 5, 400, 40
    x, ig, rg, dout = (rnd(k, b, n, d, dtype=dtype) for k in range(4))
    decay, dfin = rnd(5, d).abs(), rnd(7, b, d)
    dfin[:, 3], dfin[:, 5] = float("inf"), -float("inf")
    ln = torch.zeros(b, dtype=torch.int32, device="cuda")
    s = sq.gated_recurrence(x, ig, rg, decay, lengths=ln, save_states=True).states
    g = sq.gated_recurrence_backward(dout, x, ig, rg, decay, s, lengths=ln, dfinal_state=dfin)
    assert torch.equal(g.dinitial_state, dfin)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_negative_decay_is_nan(dtype):
    """sqrt(1 - a^2) of a factor above 1 does not exist: its channel is NaN, no other."""
    b, n, d = 3, 100, 40
    x, ig, rg, dout = (rnd(k, b, n, d, dtype=dtype) for k in range(4))
    decay, h = rnd(5, d).abs() + 0.01, rnd(6, b, d)
    bad = decay.clone()
    bad[7], bad[20] = -0.5, -float("inf")
    ln = torch.tensor([n, 40, 0], dtype=torch.int32, device="cuda")
    r = [sq.gated_recurrence(x, ig, rg, v, initial_state=h, lengths=ln, save_states=True) for v in (decay, bad)]
    g = [sq.gated_recurrence_backward(dout, x, ig, rg, v, q.states, lengths=ln) for v, q in zip((decay, bad), r)]
    rest = [c for c in range(d) if c not in (7, 20)]
    for u, v in zip((*r[0], *g[0]), (*r[1], *g[1])):
        within(v[..., rest], u[..., rest].double(), 2 * (20 + 10 * n) * EPS * u.abs().max().item())
    for c in (7, 20):
        for v in (r[1].out, g[1].dx, g[1].dinput_gate, g[1].drecurrence_gate):
            assert torch.isnan(v[0, :, c]).all() and torch.isnan(v[1, :40, c]).all()
            assert not v[1, 40:, c].any() and not v[2, :, c].any()
        assert torch.isnan(r[1].final_state[:2, c]).all() and r[1].final_state[2, c] == h[2, c]
        assert torch.isnan(g[1].ddecay[c])
    step = [v[:, 0].contiguous() for v in (x, ig, rg)]
    y = sq.gated_recurrence_step(*step, bad, h.clone())
    assert torch.isnan(y).any(0).tolist() == [c in (7, 20) for c in range(d)]


# ---------------------------------------------------------------- logits near float32's ends

@pytest.mark.parametrize("dtype", [F32, torch.bfloat16])
@pytest.mark.parametrize("tokens", [3, 40, 300])
def test_loss_of_logits_near_the_largest(tokens, dtype):
    """Logits of 3e38 are finite, their multiples by log2 e are not. A row's lse is its
    largest logit then (its spacing in float32 is 2^104), the softmax 1 there."""
    big = 2.0 ** 64
    x = torch.zeros(tokens, 16, device="cuda", dtype=dtype)
    w = torch.zeros(700, 16, device="cuda", dtype=dtype)
    kind = torch.arange(tokens, device="cuda") % 3
    t = (torch.arange(tokens, device="cuda") * 37 + 1) % 700
    x[kind == 0, 0] = big            # word 5 is far above all others
    w[5, 0] = 0.75 * big
    x[kind == 1, 1] = big            # all words near the lowest, word 9 a little less so
    w[:, 1] = -0.875 * big
    w[9, 1] = -0.75 * big
    x[kind == 2, 2] = 1.0            # an ordinary row among them
    w[:, 2] = torch.arange(700, device="cuda").to(dtype) / 256
    logits = x.double() @ w.double().t()
    lse = torch.logsumexp(logits, 1)
    at = torch.arange(tokens, device="cuda")
    loss = lse - logits[at, t]
    for targets in (t, logits.argmax(1)):
        loss = lse - logits[at, targets]
        r = sq.linear_cross_entropy(x, w, targets)
        within(r.lse, lse, 32 * EPS * lse.abs(), "lse")
        within(r.loss, loss, 64 * EPS * (1 + lse.abs()) * (kind == 2).double(), "loss")
        d = torch.ones(tokens, device="cuda")
        g = sq.linear_cross_entropy_backward(d, x, w, targets, r.lse)
        p = torch.softmax(logits, 1)
        size = p.clone()
        size[at, targets] += 1
        p[at, targets] -= 1
        # G is rounded to 16 bits for 16-bit types, its exponentials' arguments to lse's spacing
        u = U[dtype] + 64 * EPS * (1 + logits.abs().amax(1)[kind == 2].max())
        err = u * size + 2.0 ** -126
        for got, ref, e in ((g.dx, p @ w.double(), err @ w.double().abs()),
                            (g.dweight, p.t() @ x.double(), err.t() @ x.double().abs())):
            within(got, ref, 2 * e)


@pytest.mark.parametrize("dtype", [F32, torch.bfloat16])
@pytest.mark.parametrize("tokens", [3, 40, 300])
def test_far_logits_change_no_other_row(tokens, dtype):
    """A row's loss does not depend on what lies in its neighbours."""
    x, w, t = loss_case(tokens, 24, 500, dtype, 0.0)
    w[:, 23] = 0
    w[7, 23] = 2.0 ** 64
    x[:, 23] = 0
    want = sq.linear_cross_entropy(x, w, t)
    far = torch.arange(tokens, device="cuda") % 3 == 1
    x[far, 23] = 0.75 * 2.0 ** 64
    got = sq.linear_cross_entropy(x, w, t)
    assert (got.lse[far] > 2e38).all()
    assert torch.equal(got.lse[~far], want.lse[~far]) and torch.equal(got.loss[~far], want.loss[~far])


# ---------------------------------------------------------------- long sums

@pytest.mark.parametrize("tokens,width,vocab,masked", [(65536, 64, 256, 0.0), (50001, 40, 77, 0.4),
                                                       (20000, 256, 9600, 0.0), (12345, 30, 1001, 1.0)])
def test_weights_gradient_over_many_tokens(tokens, width, vocab, masked):
    """In float32 dW is a sum over tokens, of either sign: n of them one after the other
    are off by 0.6 sqrt(n / 2) units of 2^-24 at random (each addition rounds a partial
    sum of sqrt(k) terms by 0.3 units of its size at most, twice that for the spread of
    sizes). No chain is longer than 1024, whose sums are added; 8 units for the terms."""
    x, w = rnd(1, tokens, width), rnd(2, vocab, width, std=1.5 / width ** 0.5)
    g = torch.Generator().manual_seed(3)
    t = torch.randint(vocab, (tokens,), generator=g)
    t[torch.rand(tokens, generator=g) < masked] = -100
    t = t.cuda()
    d = torch.full((tokens,), 1.0 / tokens, device="cuda")
    r = sq.linear_cross_entropy(x, w, t)
    got = sq.linear_cross_entropy_backward(d, x, w, t, r.lse)
    want = torch.zeros(vocab, width, dtype=torch.float64, device="cuda")
    for i in range(0, tokens, 4096):
        xs, ts = x[i:i + 4096][t[i:i + 4096] >= 0].double(), t[i:i + 4096][t[i:i + 4096] >= 0]
        p = torch.softmax(xs @ w.double().t(), 1)
        p[torch.arange(len(ts), device="cuda"), ts] -= 1
        want += p.t() @ xs / tokens
    if masked == 1.0:
        assert not got.dweight.any() and not got.dx.any()
        return
    units = 0.6 * (1024 / 2) ** 0.5 + 0.6 * (tokens / 1024 / 2) ** 0.5 + 8
    assert ((got.dweight.double() - want).norm() / want.norm()).item() <= units * EPS
    again = sq.linear_cross_entropy_backward(d, x, w, t, r.lse)
    assert torch.equal(again.dweight, got.dweight) and torch.equal(again.dx, got.dx)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens,width,vocab,masked", [(400000, 64, 100, 0.0), (100000, 40, 300, 0.4),
                                                       (70000, 24, 9000, 0.0), (5000, 72, 200, 0.9),
                                                       (3000, 16, 70, 1.0)])
def test_weights_gradient_over_many_tokens_in_16_bits(tokens, width, vocab, masked, dtype):
    """Rounding G and the outputs: 0.65 u (below). The tensor cores cut off each of a chain's
    n / 16 additions by half a unit of 2^-23 on average, of a sum of sqrt(k) terms: n / 24
    units of 2^-24 at its end, 0.17 u of float16 for the 32768 tokens that a chain has."""
    x, w, t = loss_case(tokens, width, vocab, dtype, masked)
    d = torch.full((tokens,), (1024.0 if dtype == torch.float16 else 1.0) / tokens, device="cuda")
    r = sq.linear_cross_entropy(x, w, t)
    got = sq.linear_cross_entropy_backward(d, x, w, t, r.lse)
    want = torch.zeros(vocab, width, dtype=torch.float64, device="cuda")
    ok = (t >= 0) & (t < vocab)
    for i in range(0, tokens, 8192):
        xs, ts = x[i:i + 8192][ok[i:i + 8192]].double(), t[i:i + 8192][ok[i:i + 8192]]
        p = torch.softmax(xs @ w.double().t(), 1)
        p[torch.arange(len(ts), device="cuda"), ts] -= 1
        want += p.t() @ xs * d[0].double()
    if masked == 1.0:
        assert not got.dweight.any() and not got.dx.any()
        return
    assert ((got.dweight.double() - want).norm() / want.norm()).item() <= 0.82 * U[dtype]
    again = sq.linear_cross_entropy_backward(d, x, w, t, r.lse)
    assert torch.equal(again.dweight, got.dweight) and torch.equal(again.dx, got.dx)


# ---------------------------------------------------------------- dropout's words

@pytest.mark.parametrize("seed,offset", [
    (0, 0), (2 ** 64 - 1, 2 ** 64 - 1), (0x299F31D0A4093822, 0x0370734413198A2E),
    (1 << 32, 0), (0, 1 << 32), (0x80000000, 0x8000000080000000)])
def test_dropout_follows_the_generator(seed, offset):
    """All bits of seed and offset reach the words (test_training_edges.py pins these by
    published vectors): masks of several chances bound each word from both sides."""
    n = 4096
    want = torch.tensor(words(0, n, seed, offset))
    x = torch.ones(n, device="cuda")
    signed = lambda v: v - 2 ** 64 if v >= 2 ** 63 else v
    for p in (0.001, 0.1, 0.25, 0.5, 0.75, 0.999):
        keep = want >= int(p * 2 ** 32)
        for s in (seed, torch.tensor([signed(seed)], device="cuda")):
            assert torch.equal((sq.dropout(x, p, s, offset=signed(offset)) != 0).cpu(), keep)
            assert torch.equal((sq.dropout_backward(x, p, s, offset=signed(offset)) != 0).cpu(), keep)


# ---------------------------------------------------------------- far and long recurrences

def test_recurrence_gradients_beyond_2_31_values():
    """The end of an array of more than 2^31 values: gradients flow from the end, so those
    of the last 100 steps differ from a short call's by what its start does not know,
    e^-0.45 a step over 400 of them."""
    n, d = 2 ** 21 + 100, 1040
    g = torch.Generator(device="cuda").manual_seed(1)
    new = lambda: torch.empty(1, n, d, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    x, ig, dout = new(), new(), new()
    rg = torch.zeros(1, 1, 1, device="cuda", dtype=torch.bfloat16).expand(1, n, d).contiguous()
    decay = torch.full((d,), 0.9, device="cuda")
    s = sq.gated_recurrence(x, ig, rg, decay, save_states=True).states
    whole = sq.gated_recurrence_backward(dout, x, ig, rg, decay, s)
    end = slice(n - 500, n)
    part = [v[:, end].contiguous() for v in (x, ig, rg)]
    s = sq.gated_recurrence(*part, decay, save_states=True).states
    tail = sq.gated_recurrence_backward(dout[:, end].contiguous(), *part, decay, s)
    for name in ("dx", "dinput_gate", "drecurrence_gate"):
        a, b = getattr(whole, name)[:, -100:], getattr(tail, name)[:, -100:].double()
        # memories of 1 / (1 - e^-0.45) < 3 steps: 4 (20 + 10 * 3) units of the largest, and
        # two roundings to bfloat16
        within(a, b, 2.0 ** -8 * b.abs() + 4 * 50 * EPS * b.abs().max().item())
    # ddecay: the other steps' part is missing from the short call's, n / 500 times as much
    assert torch.isfinite(whole.ddecay).all()


def test_recurrence_gradients_of_a_long_memory_in_float32():
    """Factors up to 0.9999 over 4000 steps: neither states nor their gradients add up
    errors in one direction. Each is off by sqrt(n) units at random, of which four times
    are allowed, and what a gradient multiplies them with by 20 units."""
    n, d = 4000, 64
    x, ig, dout = rnd(1, 1, n, d), rnd(2, 1, n, d), rnd(4, 1, n, d)
    rg = rnd(3, 1, n, d, std=0.1)
    decay = torch.logspace(-3.7, -0.5, d, device="cuda")
    wide = [v.double().requires_grad_() for v in (x, ig, rg, decay)]
    out, _ = ref_recurrence(*wide, None, None)
    want = torch.autograd.grad((out * dout.double()).sum(), wide)
    s = sq.gated_recurrence(x, ig, rg, decay, save_states=True).states
    got = sq.gated_recurrence_backward(dout, x, ig, rg, decay, s)
    with torch.no_grad():
        xd, i, r = x.double(), torch.sigmoid(ig.double()), torch.sigmoid(rg.double())
        la = -decay.double() * r
        a, root = torch.exp(la), torch.sqrt(-torch.expm1(2 * la))
        grad, later = torch.empty_like(xd), torch.zeros(1, d, dtype=torch.float64, device="cuda")
        for t in range(n - 1, -1, -1):
            grad[:, t] = dout[:, t].double() + later
            later = a[:, t] * grad[:, t]
        top = grad.abs().amax(1)                      # of a channel
        states = out.abs().amax(1)
        off = (4 * n ** 0.5 + 20) * EPS
        term = (r * a * (states + a / root * i * xd.abs())).amax(1)     # of ddecay, per G
        size = {"dx": (root * i).amax(1), "dinput_gate": (root * xd.abs() * i * (1 - i)).amax(1),
                "drecurrence_gate": 2 * term * decay.double() / 2}
    for name, w in zip(("dx", "dinput_gate", "drecurrence_gate"), want):
        err = (getattr(got, name).double() - w).abs().amax(1)
        assert (err <= off * top * size[name] + U[F32] * w.abs().amax(1)).all(), name
    # ddecay: n terms with both errors, those of neighbours alike for a memory's length
    err = (got.ddecay.double() - want[3]).abs()
    assert (err <= 2 * off * n * (top * term)[0]).all()


# ---------------------------------------------------------------- the loss's rounding in 16 bits

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens,width,vocab", [(777, 256, 3000), (4096, 64, 256), (40, 128, 1000), (900, 100, 70)])
def test_loss_gradients_round_twice_in_16_bits(tokens, width, vocab, dtype):
    """The logits' gradients are rounded to 16 bits between the products, with weights that
    differ from token to token: a random relative error of u sqrt(E[1 / m^2] / 3) = 0.425 u
    over mantissas m in [1, 2), as much as rounding the outputs leaves; both together
    0.425 sqrt(2) u = 0.6 u, and 0.05 u for mantissas that do not spread evenly."""
    x, w, t = loss_case(tokens, width, vocab, dtype, 0.0)
    d = rnd(9, tokens).abs() + 0.1
    r = sq.linear_cross_entropy(x, w, t)
    g = sq.linear_cross_entropy_backward(d, x, w, t, r.lse)
    p = torch.softmax(x.double() @ w.double().t(), 1)
    p[torch.arange(tokens, device="cuda"), t] -= 1
    p *= d.double()[:, None]
    for got, ref in ((g.dx, p @ w.double()), (g.dweight, p.t() @ x.double())):
        assert ((got.double() - ref).norm() / ref.norm()).item() <= 0.65 * U[dtype]


# ---------------------------------------------------------------- two callers at once

def test_two_threads_call_at_once():
    """Calls of two host threads, each on a stream of its own, do not share workspaces."""
    jobs = []
    for seed in (0, 50):
        x, ig, rg, dout = (rnd(seed + k, 2, 900, 96, dtype=torch.bfloat16) for k in range(4))
        decay = rnd(seed + 4, 96).abs()
        lx, lw, lt = loss_case(300, 100, 2001, torch.bfloat16, 0.2, seed=seed)
        fx, fw, ft = loss_case(3000, 40, 77, F32, 0.2, seed=seed)

        def job(stream=None, x=x, ig=ig, rg=rg, dout=dout, decay=decay, lx=lx, lw=lw, lt=lt, fx=fx, fw=fw, ft=ft):
            k = {"stream": stream}
            r = sq.gated_recurrence(x, ig, rg, decay, save_states=True, **k)
            g = sq.gated_recurrence_backward(dout, x, ig, rg, decay, r.states, **k)
            out = [*r, *g, sq.dropout(lx, 0.3, 5, **k)]
            for a, b, t in ((lx, lw, lt), (fx, fw, ft)):
                l = sq.linear_cross_entropy(a, b, t, **k)
                out += [*l, *sq.linear_cross_entropy_backward(torch.ones_like(l.loss), a, b, t, l.lse, **k)]
            return out

        jobs.append(job)
    want = [job() for job in jobs]
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        s = torch.cuda.Stream()
        for _ in range(10):
            got[i].append(jobs[i](stream=s))
        s.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    for i in range(2):
        assert len(got[i]) == 10
        for out in got[i]:
            for a, b in zip(out, want[i]):
                assert torch.equal(a, b)


# ---------------------------------------------------------------- wide rows

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens,width,vocab", [(30, 4096, 256), (60, 5000, 300), (1000, 4096, 256), (300, 10000, 500),
                                                (200, 2112, 1000), (5, 30000, 77)])
def test_loss_of_wide_rows_keeps_float32(tokens, width, vocab, dtype):
    """A chain of n additions on the tensor cores shrinks its sum by n 1.5e-8 (they cut off);
    none has more than 64, so logits are off by 1e-6 of their size, and lse and loss,
    which are larger here, by less."""
    x, w, t = loss_case(tokens, width, vocab, dtype, 0.0)
    r = sq.linear_cross_entropy(x, w, t)
    logits = x.double() @ w.double().t()
    lse = torch.logsumexp(logits, 1)
    loss = lse - logits[torch.arange(tokens, device="cuda"), t]
    for got, ref in ((r.lse, lse), (r.loss, loss)):
        assert ((got.double() - ref).norm() / ref.norm()).item() <= 1e-6

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_loss_gradient_refuses_rows_too_wide_for_16_bits(dtype):
    """Rows beyond 2^16 values: the loss in parts of 64 additions, each cut off by a unit of
    2^-23 at most, and a rounded sum for each part: below 512 units of 2^-24 of the largest
    partial sum (within 4 times the logits' size). The gradient does not take them."""
    n = (1 << 16) + 8
    x, w = rnd(1, 3, n, dtype=dtype), rnd(2, 5, n, dtype=dtype, std=2.0 ** -8)
    t = torch.tensor([0, 4, 2], device="cuda")
    r = sq.linear_cross_entropy(x, w, t)
    logits = x.double() @ w.double().t()
    off = 4 * 512 * EPS * logits.abs().amax(1)
    within(r.lse, torch.logsumexp(logits, 1), off)
    within(r.loss, torch.logsumexp(logits, 1) - logits[torch.arange(3, device="cuda"), t], 2 * off)
    with pytest.raises(ValueError, match="width must be at most 2.16 in 16-bit types"):
        sq.linear_cross_entropy_backward(torch.ones(3, device="cuda"), x, w, t, r.lse)
    sq.linear_cross_entropy_backward(torch.ones(3, device="cuda"), x[:, :-8], w[:, :-8], t, r.lse)
    dev = capi.DeviceHandle(0)
    block = capi.SEQ_SIGNATURES["ferrum_linear_cross_entropy_bwd"]
    args = block(struct_size=ctypes.sizeof(block), dtype=1, tokens=1, width=n, vocab=1)
    assert capi.lib().ferrum_linear_cross_entropy_bwd(dev.ptr, ctypes.byref(args), None) == capi.FERRUM_ERR_INVALID_ARG
    assert "2^16" in capi.last_error()
