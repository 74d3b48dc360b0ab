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
