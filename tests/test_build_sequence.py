"""The build step of the module on torch tensors: left out where torch is not
installed, repeated for another version of torch."""

from __future__ import annotations

import importlib.util
import os

import pytest

from conftest import PKG_DIR


@pytest.fixture
def build(tmp_path, monkeypatch):
    spec = importlib.util.spec_from_file_location("build_py", os.path.join(PKG_DIR, "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    commands = []
    monkeypatch.setattr(mod, "BUILD", str(tmp_path))
    monkeypatch.setattr(mod, "_run", commands.append)
    monkeypatch.setattr(mod, "_stale", lambda target, deps: False)
    mod.commands = commands
    return mod


def test_without_torch_the_rest_is_built(build, monkeypatch, capsys):
    monkeypatch.setattr(build, "_torch_version", lambda: None)
    assert build.build_sequence() is False
    build.build(jobs=1, force=True)
    targets = [c[c.index("-o") + 1] for c in build.commands]
    assert build.LIB in targets and build.EXT in targets and build.SEQ_EXT not in targets
    assert "torch is not installed" in capsys.readouterr().err


def test_another_torch_rebuilds_it(build, monkeypatch):
    for version, count in (("2.0", 1), ("2.0", 1), ("2.1", 2), ("2.1", 2)):
        monkeypatch.setattr(build, "_torch_version", lambda: version)
        assert build.build_sequence() is True
        assert len(build.commands) == count


def test_a_failed_build_is_tried_again(build, monkeypatch):
    monkeypatch.setattr(build, "_torch_version", lambda: "2.0")

    def fail(cmd):
        raise RuntimeError("command failed")

    monkeypatch.setattr(build, "_run", fail)
    with pytest.raises(RuntimeError):
        build.build_sequence()
    monkeypatch.setattr(build, "_run", build.commands.append)
    assert build.build_sequence() is True and len(build.commands) == 1
