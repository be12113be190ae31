"""The library and the module of native calls are built apart: what the module needs and is not there (a host compiler,
Python's or torch's headers) does not keep the library from being built and used (on the CPU)."""

from __future__ import annotations

import sys

import pytest
import torch

from omniwave_amd import _build, _native, cross_entropy_hip, norms, rms_norm_hip


@pytest.fixture
def small_build(monkeypatch, tmp_path):
    monkeypatch.setattr(_build, "SOURCES", ["route.cpp"])
    monkeypatch.setattr(_build, "LIB_PATH", tmp_path / "libomniwave_amd.so")
    monkeypatch.setattr(_build, "GLUE_PATH", tmp_path / "_glue.so")
    return tmp_path


@pytest.mark.parametrize("missing", ["compiler", "headers", "libraries", "torch"])
def test_a_module_that_cannot_be_built(small_build, monkeypatch, missing) -> None:
    def commands(obj, out, lib_dir):
        if missing == "torch":
            raise ImportError("No module named 'torch'")
        fail = [sys.executable, "-c", "raise SystemExit('Python.h: No such file or directory')"]
        fine = [sys.executable, "-c", "pass"]
        if missing == "compiler":
            return ["/nowhere/g++"], ["/nowhere/g++"]
        return (fail, fine) if missing == "headers" else (fine, fail)

    monkeypatch.setattr(_build, "glue_commands", commands)
    (small_build / "_glue.so").write_bytes(b"of an earlier build")
    with pytest.warns(RuntimeWarning, match="_glue.so"):
        assert _build.build() == small_build / "libomniwave_amd.so"
    assert (small_build / "libomniwave_amd.so").stat().st_size > 1000
    assert not (small_build / "_glue.so").exists()  # it belonged to another library


def test_a_library_that_cannot_be_built_leaves_the_old_one(small_build, monkeypatch) -> None:
    (small_build / "libomniwave_amd.so").write_bytes(b"old")
    monkeypatch.setattr(_build, "SOURCES", ["nothing.cpp"])
    monkeypatch.setattr(_build, "glue_commands", lambda *a: ([sys.executable, "-c", "pass"],) * 2)
    with pytest.raises(RuntimeError, match="build failed"):
        _build.build()
    assert (small_build / "libomniwave_amd.so").read_bytes() == b"old"


def test_the_operators_need_the_library_alone(monkeypatch) -> None:
    monkeypatch.setattr(_native, "_glue", None)
    monkeypatch.setattr(_native, "_glue_error", "cannot load _glue.so")
    x = torch.zeros(2, 8)
    assert "not on a GPU" in norms.gpu_reason(x)
    for call in (lambda: rms_norm_hip(x, torch.ones(8)), lambda: cross_entropy_hip(x, torch.zeros(2, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="not on a GPU"):
            call()
