"""The example model trains on the sequence operators and decodes token by
token to the same logits."""

from __future__ import annotations

import importlib.util
import math
import os

import pytest

from conftest import REPO, gpu_available


@pytest.mark.gpu
def test_sequence_block_trains_and_decodes():
    if not gpu_available():
        pytest.skip("no B200")
    spec = importlib.util.spec_from_file_location(
        "sequence_block", os.path.join(REPO, "examples", "sequence_block.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    losses, gap = mod.main(steps=120)
    # learning at all needs every gradient; the loss starts at ln(16) = 2.77
    assert losses[-1] < 0.7 * math.log(16)
    # float32 through two layers: products of 64 and 96 terms, a scan of 96 steps
    assert gap < 1e-4
