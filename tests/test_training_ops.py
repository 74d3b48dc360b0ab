"""Gated recurrence, dropout and the loss, CPU part: argument blocks against the
header, bad arguments refused by name before any GPU work."""

from __future__ import annotations

import ctypes
import subprocess

import pytest
import torch

from conftest import REPO

from ferrum_gpu import capi, sequence as sq

X, W, G = torch.zeros(2, 3, 4), torch.zeros(4), torch.zeros(2, 4)
T = torch.zeros(2, 3, dtype=torch.int64)


def test_argument_blocks_match_the_header(tmp_path):
    """Size and every field offset, as the C compiler lays them out."""
    blocks = {"ferrum_recurrence_args": capi.RecurrenceArgs,
              "ferrum_dropout_args": capi.DropoutArgs,
              "ferrum_cross_entropy_args": capi.CrossEntropyArgs}
    lines, want = [], []
    for c, py in blocks.items():
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        lines += [f'printf("%zu\\n", offsetof({c}, {f}));' for f, _ in py._fields_]
        want.append(ctypes.sizeof(py))
        want += [getattr(py, f).offset for f, _ in py._fields_]
    src = tmp_path / "o.c"
    src.write_text('#include <stdio.h>\n#include "ferrum_seq.h"\nint main(void) {'
                   + "\n".join(lines) + "return 0; }")
    exe = str(tmp_path / "o")
    subprocess.run(["gcc", f"-I{REPO}/include", str(src), "-o", exe], check=True)
    got = subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()
    assert [int(v) for v in got] == want


@pytest.mark.parametrize("call", [
    lambda: sq.gated_recurrence(X, X, X, W),
    lambda: sq.gated_recurrence_backward(X, X, X, X, W, X),
    lambda: sq.gated_recurrence_step(G, G, G, W, G),
    lambda: sq.dropout(X, 0.1, 3),
    lambda: sq.dropout_backward(X, 0.1, 3),
    lambda: sq.linear_cross_entropy(X, G, T),
    lambda: sq.linear_cross_entropy_backward(T, X, G, T, T),
])
def test_cpu_tensors_are_refused(call):
    with pytest.raises(ValueError, match="must be a CUDA tensor"):
        call()


@pytest.mark.parametrize("match,call", [
    ("decay must be a CUDA tensor, got float", lambda: sq.gated_recurrence(X, X, X, 0.5)),
    ("save_states must be a truth value, got str",
     lambda: sq.gated_recurrence(X, X, X, W, save_states="yes")),
    ("p must be a number, got str", lambda: sq.dropout(X, "0.1", 3)),
    ("p must be a number, got NoneType", lambda: sq.dropout(X, None, 3)),
    ("offset must be an integer, got float", lambda: sq.dropout(X, 0.1, 3, offset=1.5)),
    ("dtype must be a torch.dtype, got str", lambda: sq.dropout_backward(X, 0.1, 3, dtype="f32")),
    ("residual must be a CUDA tensor, got float", lambda: sq.dropout(X, 0.1, 3, residual=1.0)),
    ("targets must be a CUDA tensor, got list", lambda: sq.linear_cross_entropy(X, G, [1, 2])),
    ("x is required", lambda: sq.linear_cross_entropy(None, G, T)),
])
def test_the_argument_is_named(match, call):
    with pytest.raises(ValueError, match=match):
        call()


def test_c_entries_refuse_a_wrong_block():
    """Without a device handle nothing else of the block is looked at."""
    for name in ("ferrum_gated_recurrence", "ferrum_dropout", "ferrum_linear_cross_entropy"):
        args = capi.SEQ_SIGNATURES[name](struct_size=1)
        assert getattr(capi.lib(), name)(None, ctypes.byref(args), None) == capi.FERRUM_ERR_INVALID_ARG
