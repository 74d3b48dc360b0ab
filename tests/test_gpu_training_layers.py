"""The example's layers side by side: what several of one kind do not share."""

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


def test_layers_draw_masks_of_their_own(example):
    """Two layers of one model, alike but for their place in it, drop other values, in
    the forward and in the gradient; each draws another mask at every step."""
    torch.manual_seed(0)
    layers = [example.RecurrenceLayer(k).cuda() for k in (0, 1)]
    layers[1].load_state_dict(layers[0].state_dict())
    h = torch.randn(4, 64, example.WIDTH, device="cuda")
    dropped = []
    for _ in range(2):
        for layer in layers:
            x = h.clone().requires_grad_()
            y = layer(x)
            dropped.append((y == h).detach())
            # the gradient drew the same mask: y - h is scale's gradient times scale, both sums
            # of 256 values below 8 (512 roundings of 2^-24 times 8: 2.5e-4)
            g = torch.autograd.grad(y.sum(), layer.scale)[0]
            kept = (y - h).detach().sum((0, 1))
            assert torch.allclose(g * layer.scale.detach(), kept, rtol=0, atol=1e-3)
    n = h.numel()
    for m in dropped:                  # a share of DROP, within 6 standard deviations
        assert abs(m.sum().item() - n * example.DROP) < 6 * (n * example.DROP) ** 0.5
    for i in range(4):
        for j in range(i):             # and DROP^2 in common
            both = n * example.DROP ** 2
            assert (dropped[i] & dropped[j]).sum().item() < both + 6 * both ** 0.5
