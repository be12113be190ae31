"""Layer norm: what the call and its operators refuse, on the CPU, and the C entry points' argument checks."""

from __future__ import annotations

import ctypes

import pytest
import torch

from omniwave_amd import _native, layer_norm_hip, norms

X, W = torch.zeros(4, 10), torch.ones(10)


@pytest.mark.parametrize("kwargs,text", [
    (dict(x=X.double()), "dtype"),
    (dict(x=torch.zeros(())), "scalar"),
    (dict(x=torch.zeros(2, 8193)), "8192"),
    (dict(weight=W[:9]), "weight"),
    (dict(weight=W[None]), "weight"),
    (dict(weight=W.int()), "weight"),
    (dict(bias=W.double()), "bias"),
    (dict(bias=torch.ones(11)), "bias"),
    (dict(bias=torch.ones(10, device="meta")), "bias"),
    (dict(eps=-1e-6), "eps"),
    (dict(eps=float("nan")), "eps"),
    (dict(eps=float("inf")), "eps"),
])
def test_refusals(kwargs, text) -> None:
    args = {"x": X, "weight": W, "bias": W, **kwargs}
    with pytest.raises(ValueError, match=text):
        layer_norm_hip(args.pop("x"), args.pop("weight"), args.pop("bias"), **args)


def test_the_cpu_has_no_kernel() -> None:
    for args in ((X,), (X, W), (X, W, W), (X, None, W)):
        with pytest.raises(RuntimeError, match="not supported"):
            layer_norm_hip(*args)
    ops = torch.ops.omniwave_amd
    with pytest.raises(RuntimeError, match="not supported"):
        ops.layer_norm_fwd(X, W, W, 1e-6)
    with pytest.raises(RuntimeError, match="not supported"):
        ops.layer_norm_bwd(X, X, W, W, 1e-6, [True] * 3)


@pytest.fixture
def launches(monkeypatch):
    calls = []
    monkeypatch.setattr(norms, "_on", lambda *args: calls.append(args))
    monkeypatch.setattr(norms, "gpu_reason", lambda t: None)

    class Anywhere:
        def __init__(self, device):
            pass

        def __enter__(self):
            pass

        def __exit__(self, *args):
            pass

    monkeypatch.setattr(torch.cuda, "device", Anywhere)
    return calls


@pytest.mark.parametrize("bad", [dict(x=X[:, :9]), dict(x=X.double()), dict(weight=W[:9]), dict(bias=W.int()),
                                 dict(weight=torch.ones(10, device="meta"))])
def test_what_the_operators_get(launches, bad) -> None:
    t = {"x": X, "weight": W, "bias": W, **bad}
    with pytest.raises(ValueError):
        norms._run_layer_norm_forward(*t.values(), 1e-6)
    with pytest.raises(ValueError):
        norms._run_layer_norm_backward(torch.zeros_like(t["x"]), *t.values(), 1e-6, [True] * 3)
    assert not launches


@pytest.mark.parametrize("up", [torch.zeros(4, 9), torch.zeros(40), X.bfloat16(), torch.zeros(4, 10, device="meta")])
def test_upstream_gradients(launches, up) -> None:
    with pytest.raises(ValueError, match="upstream"):
        norms._run_layer_norm_backward(up, X, W, W, 1e-6, [True] * 3)
    assert not launches
    norms._run_layer_norm_backward(X, X, W, W, 1e-6, [True] * 3)
    norms._run_layer_norm_backward(X, X, W, W, 1e-6, [False] * 3)  # nothing is asked for
    norms._run_layer_norm_forward(X, W, W, 1e-6)
    assert len(launches) == 2


def test_c_entry_points_check_their_arguments() -> None:
    lib, p = _native.lib(), ctypes.c_void_p(256)

    def desc(**kw):
        d = _native.OwLayerNorm(rows=4, x_stride=10, x=256, weight=256, bias=256, channels=10, dtype=0, weight_dtype=0,
                                bias_dtype=0, eps=1e-6)
        for k, v in kw.items():
            setattr(d, k, v)
        return ctypes.byref(d)

    def refused(rc, text, code=1):
        assert rc == code and text in lib.ow_last_error(), lib.ow_last_error()

    refused(lib.ow_layer_norm_fwd(None, p, None), b"NULL")
    refused(lib.ow_layer_norm_fwd(desc(dtype=7), p, None), b"dtype", 2)
    refused(lib.ow_layer_norm_fwd(desc(rows=-1), p, None), b"negative")
    refused(lib.ow_layer_norm_fwd(desc(channels=8193), p, None), b"8192", 2)
    refused(lib.ow_layer_norm_fwd(desc(rows=1 << 31), p, None), b"2^31", 2)
    refused(lib.ow_layer_norm_fwd(desc(x=None), p, None), b"NULL")
    refused(lib.ow_layer_norm_fwd(desc(weight_dtype=9), p, None), b"dtype")
    refused(lib.ow_layer_norm_fwd(desc(), None, None), b"NULL")
    assert lib.ow_layer_norm_fwd(desc(rows=0), None, None) == 0 and lib.ow_layer_norm_fwd(desc(channels=0), None, None) == 0
    assert lib.ow_layer_norm_bwd_workspace(None) == 0 and lib.ow_layer_norm_bwd_workspace(desc(rows=1)) == 0
    big = desc(rows=100000)
    assert lib.ow_layer_norm_bwd_workspace(big) >= 4 * 2 * 10 * 2
    refused(lib.ow_layer_norm_bwd(desc(rows=0), p, 10, p, p, p, None, 0, None), b"no rows")
    refused(lib.ow_layer_norm_bwd(desc(), None, 10, p, p, p, None, 0, None), b"NULL")
    refused(lib.ow_layer_norm_bwd(desc(weight=None), p, 10, p, p, p, None, 0, None), b"not given")
    refused(lib.ow_layer_norm_bwd(big, p, 10, p, p, p, p, 8, None), b"workspace")
    refused(lib.ow_layer_norm_bwd(big, p, 10, p, p, p, ctypes.c_void_p(257), 1 << 30, None), b"workspace")
