"""Sequence operators, CPU part: the binding mirrors include/ferrum_seq.h, the
library exports it, and bad arguments are refused before any GPU work."""

from __future__ import annotations

import ctypes
import os
import re
import subprocess

import pytest
import torch

from conftest import REPO

from ferrum_gpu import capi, sequence as sq

HEADER = os.path.join(REPO, "include", "ferrum_seq.h")


def test_header_and_binding_agree():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    assert sorted(set(re.findall(r"\b(ferrum_[a-z0-9_]+)\s*\(", text))) == sorted(capi.SEQ_SIGNATURES)
    for name in capi.SEQ_SIGNATURES:
        assert hasattr(capi.lib(), name)


def test_argument_blocks_match_the_header(tmp_path):
    """Size and every field offset, as the C compiler lays them out."""
    blocks = {"ferrum_conv1d_args": capi.ConvArgs, "ferrum_scan_args": capi.ScanArgs,
              "ferrum_norm_args": capi.NormArgs, "ferrum_long_conv_args": capi.LongArgs}
    lines = []
    for c, py in blocks.items():
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        lines += [f'printf("%zu\\n", offsetof({c}, {f}));' for f, _ in py._fields_]
    src = tmp_path / "o.c"
    src.write_text('#include <stdio.h>\n#include "ferrum_seq.h"\nint main(void) {'
                   + "\n".join(lines) + "return 0; }")
    exe = str(tmp_path / "o")
    subprocess.run(["gcc", f"-I{REPO}/include", str(src), "-o", exe], check=True)
    got = [int(v) for v in subprocess.run([exe], check=True, capture_output=True,
                                          text=True).stdout.split()]
    want = []
    for py in blocks.values():
        want.append(ctypes.sizeof(py))
        want += [getattr(py, f).offset for f, _ in py._fields_]
    assert got == want


@pytest.mark.parametrize("name", sorted(capi.SEQ_SIGNATURES))
def test_null_device_and_block_are_refused(name):
    args = capi.SEQ_SIGNATURES[name]()
    assert getattr(capi.lib(), name)(None, ctypes.byref(args), None) == capi.FERRUM_ERR_INVALID_ARG
    assert "device handle" in capi.last_error()


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 3, 4)
    with pytest.raises(ValueError, match="must be a CUDA tensor"):
        sq.causal_conv1d(x, torch.zeros(4, 2))
    with pytest.raises(ValueError, match="must be a CUDA tensor"):
        sq.selective_scan(x, x, torch.zeros(4, 2), x, x)
    with pytest.raises(ValueError, match="must be a CUDA tensor"):
        sq.norm_before(x, torch.zeros(4))
    with pytest.raises(ValueError, match="must be a CUDA tensor"):
        sq.norm_after(x, torch.zeros(4))
    with pytest.raises(ValueError, match="must be a CUDA tensor"):
        sq.long_conv(x, torch.zeros(3, 4))
    with pytest.raises(ValueError, match="x is required"):
        sq.long_conv(None, torch.zeros(3, 4))
    with pytest.raises(ValueError, match="CUDA tensor"):
        sq.long_conv(x.numpy(), torch.zeros(3, 4))
    with pytest.raises(ValueError, match="CUDA tensor"):
        sq.long_conv("x", torch.zeros(3, 4))
