"""Arguments of a wrong type are refused by name, before any GPU work."""

from __future__ import annotations

import inspect

import numpy as np
import pytest
import torch

from ferrum_gpu import _sequence, sequence as sq

X, W = torch.zeros(2, 3, 4), torch.zeros(4)


@pytest.mark.parametrize("match,call", [
    ("groups must be an integer, got float", lambda: sq.norm_after(X, W, groups=1.5)),
    ("eps must be a number, got str", lambda: sq.norm_before(X, W, eps="x")),
    ("kind must be a string, got NoneType", lambda: sq.norm_after(X, W, kind=None)),
    ("gate_inside must be a truth value, got str", lambda: sq.norm_after(X, W, gate_inside="no")),
    ("activation must be None or a string, got bool",
     lambda: sq.causal_conv1d(X, W, activation=True)),
    ("delta_softplus must be a truth value, got str",
     lambda: sq.selective_scan(X, X, W, X, X, delta_softplus="yes")),
    ("weight must be a CUDA tensor, got list", lambda: sq.causal_conv1d(X, [1.0, 2.0])),
    ("positions must be a CUDA tensor, got int", lambda: sq.long_conv_step(X, X, 3, W)),
    ("CUDA tensor .got one on the host", lambda: sq.long_conv(np.zeros((2, 3, 4)), W)),
])
def test_the_argument_is_named(match, call):
    with pytest.raises(ValueError, match=match):
        call()


def test_the_binding_takes_as_many_arguments():
    """The names in refusals count on the binding's arguments being the public
    function's."""
    for name in (n for n in dir(_sequence) if not n.startswith("_")):
        count = len(inspect.signature(getattr(sq, name)).parameters)
        for n in (count - 1, count + 1):
            with pytest.raises(TypeError):
                getattr(_sequence, name)(*[None] * n)
