"""The test by which the sequence operators refuse outputs that share memory with
an input, against numpy's exact one."""

from __future__ import annotations

import random

import numpy as np
import pytest
import torch

from ferrum_gpu import _sequence


def shares(a, b):
    return bool(np.shares_memory(a.numpy(), b.numpy()))


def random_view(rng, base):
    """A view of 1 to 4 dimensions with any strides that stay inside `base`."""
    while True:
        dims = rng.randint(1, 4)
        size = [rng.choice([1, 2, 3, 5, 8]) for _ in range(dims)]
        stride = [rng.choice([0, 1, 2, 3, 4, 7, 12, 30, 31]) for _ in range(dims)]
        start = rng.randrange(base.numel())
        if start + sum((n - 1) * st for n, st in zip(size, stride)) < base.numel():
            return base.as_strided(size, stride, start)


@pytest.mark.parametrize("seed", range(8))
def test_random_views(seed):
    rng = random.Random(seed)
    base = torch.zeros(300)
    half = torch.zeros(0).set_(base.untyped_storage()).view(torch.float16)
    seen = set()
    for _ in range(400):
        a = random_view(rng, base)
        b = random_view(rng, base if rng.random() < 0.7 else half)
        want = shares(a, b)
        seen.add(want)
        assert _sequence._shares_memory(a, b) == want, (a.size(), a.stride(), a.storage_offset(),
                                                        b.size(), b.stride(), b.storage_offset())
    assert seen == {True, False}


def test_views_that_calls_meet():
    shares_memory = _sequence._shares_memory
    wide = torch.zeros(4, 200, 96)
    assert not shares_memory(wide[..., :32], wide[..., 32:64])       # columns of one array
    assert shares_memory(wide[..., :33], wide[..., 32:64])
    assert shares_memory(wide[:, 1:], wide[:, :-1])                  # a shifted view
    assert not shares_memory(wide[:, ::2], wide[:, 1::2])            # every other row
    assert not shares_memory(wide[..., :32].transpose(1, 2), wide[..., 32:64])
    assert shares_memory(wide.transpose(1, 2), wide[2:3, 5:6])
    assert not shares_memory(wide[:0], wide)
    assert not shares_memory(wide, torch.zeros(4, 200, 96))
    one = torch.zeros(1).expand(4, 200, 96)
    assert shares_memory(one, one[0]) and not shares_memory(one, wide)
