"""The library is built whatever becomes of the extension module."""

from __future__ import annotations

import ctypes

import pytest

from deltakv_b200 import build as B


@pytest.fixture
def small_tree(tmp_path, monkeypatch):
    csrc = tmp_path / "csrc"
    csrc.mkdir()
    (csrc / "one.cu").write_text('extern "C" int one() { return 1; }\n')
    monkeypatch.setattr(B, "CSRC", csrc)
    monkeypatch.setattr(B, "BUILD", tmp_path / "_build")
    monkeypatch.setattr(B, "LIB", tmp_path / "libone.so")
    monkeypatch.setattr(B, "STEP", tmp_path / "_step.so")
    monkeypatch.setattr(B, "STEP_SRC", csrc / "missing.cpp")
    return tmp_path


def test_library_is_linked_when_the_module_does_not_build(small_tree, monkeypatch):
    def fails():
        raise RuntimeError("g++ failed")

    monkeypatch.setattr(B, "build_step", fails)
    with pytest.raises(RuntimeError, match="g..? failed"):  # still said
        B.build()
    assert ctypes.CDLL(str(B.LIB)).one() == 1


def test_library_alone_with_a_torch_without_cuda(small_tree, monkeypatch, capsys):
    import torch

    monkeypatch.setattr(torch.version, "cuda", None)
    assert B.build() == B.LIB and ctypes.CDLL(str(B.LIB)).one() == 1
    assert not B.STEP.exists() and "not built" in capsys.readouterr().err
