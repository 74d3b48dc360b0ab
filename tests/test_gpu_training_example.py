"""The example's layers of recurrence, dropout and loss: their gradients, as
torch.autograd sees them, against the same in plain operations in 64 bits."""

from __future__ import annotations

import importlib.util
import os

import pytest
import torch

from conftest import REPO, gpu_available

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    if not gpu_available():
        pytest.skip("no B200")
    spec = importlib.util.spec_from_file_location(
        "sequence_block", os.path.join(REPO, "examples", "sequence_block.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def leaves(*shapes):
    g = torch.Generator().manual_seed(3)
    return [torch.randn(s, generator=g).cuda().requires_grad_() for s in shapes]


def same(f32, f64, terms):
    """Sums of `terms` products in float32: as many units of 2^-24, of the largest."""
    for a, b in zip(f32, f64):
        assert (a.double() - b).abs().max().item() <= 4 * terms * 2.0 ** -24 * b.abs().max().item()


def test_recurrence(example):
    b, n, d = 2, 40, 24
    ins = leaves((b, n, d), (b, n, d), (b, n, d), (d,))
    wide = [v.detach().double().requires_grad_() for v in ins]
    weights = torch.randn(b, n, d, device="cuda")
    out = example.Recurrence.apply(*ins[:3], torch.exp(ins[3]))
    x, i, r, decay = wide[0], wide[1], wide[2], torch.exp(wide[3])
    la = -decay * torch.sigmoid(r)
    h, steps = torch.zeros_like(x[:, 0]), []
    for t in range(n):
        h = torch.exp(la[:, t]) * h + torch.sqrt(-torch.expm1(2 * la[:, t])) * torch.sigmoid(i[:, t]) * x[:, t]
        steps.append(h)
    ref = torch.stack(steps, 1)
    same([out.detach()], [ref.detach()], 20 + 10 * n)
    same(torch.autograd.grad((out * weights).sum(), ins),
         torch.autograd.grad((ref * weights.double()).sum(), wide), 4 * (20 + 10 * n))


def test_dropout(example):
    x, res = leaves((5, 64), (5, 64))
    seed = torch.tensor([9], device="cuda")
    y = example.Dropout.apply(x, res, 0.25, seed)
    kept = (y - res).detach() != 0
    weights = torch.randn(5, 64, device="cuda")
    dx, dres = torch.autograd.grad((y * weights).sum(), (x, res))
    assert torch.equal(dres, weights) and not dx[~kept].any()
    same([dx], [torch.where(kept, weights.double() / 0.75, torch.zeros_like(weights).double())], 2)


def test_loss(example):
    x, w = leaves((3, 7, 32), (50, 32))
    t = torch.randint(50, (3, 7), generator=torch.Generator().manual_seed(1)).cuda()
    t[0, :3] = -100
    wide = [v.detach().double().requires_grad_() for v in (x, w)]
    loss = example.Loss.apply(x, w, t).sum() / (t >= 0).sum()
    ref = torch.nn.functional.cross_entropy((wide[0] @ wide[1].t()).view(-1, 50), t.view(-1))
    # logits of 32 products, their softmax over 50, products of 50 and 21 of those
    same([loss.detach()], [ref.detach()], 100)
    same(torch.autograd.grad(loss, (x, w)), torch.autograd.grad(ref, wide), 400)


def test_a_training_step_moves_every_parameter(example):
    """One step through all layers and operators, in training and in evaluation."""
    torch.manual_seed(0)
    model = example.Model(32).cuda()
    tokens = torch.randint(example.VOCAB, (4, 32), device="cuda")
    loss = model.loss(tokens, tokens)
    loss.backward()
    assert torch.isfinite(loss)
    for name, p in model.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all() and bool(p.grad.any()), name
    model.eval()
    with torch.no_grad():
        assert torch.equal(model.loss(tokens, tokens), model.loss(tokens, tokens))
