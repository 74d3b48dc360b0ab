"""Recurrence, dropout and the loss at their edges: clusters of blocks, decays on
both sides of the short form, infinities, sizes near a limit.

Tolerances as in test_gpu_training_ops.py, whose helpers these tests use: an
output's own rounding, and a bound in units of 2^-24 that is derived beside each
test.
"""

from __future__ import annotations

import pytest
import torch

from conftest import gpu_available
from test_gpu_training_ops import EPS, F32, TYPES, U, clean, ref_recurrence, rnd, within

from ferrum_gpu import sequence as sq

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
        within(got[~off], want[~off], (20 + 10 * min(n, 222)) * EPS * h.abs().max().clamp(min=out[~torch.isinf(out)].nan_to_num().abs().max()).item())
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
