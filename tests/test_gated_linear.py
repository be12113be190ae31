"""Gated feed-forward product: what the call and its operators refuse, on the CPU, and the C entry points' argument checks."""

from __future__ import annotations

import ctypes

import pytest
import torch

from omniwave_amd import _native, gated, gated_linear_hip

X, W, NONE = torch.zeros(2, 3, 10), torch.zeros(6, 10), torch.zeros(0)


@pytest.mark.parametrize("kwargs,text", [
    (dict(x=X.double()), "dtype"),
    (dict(x=torch.zeros(())), "scalar"),
    (dict(x=X[..., :9]), "gate_weight"),
    (dict(gate=W[:, :9]), "gate_weight"),
    (dict(gate=W[0]), "gate_weight"),
    (dict(gate=W[None]), "gate_weight"),
    (dict(up=W[:5]), "up_weight"),
    (dict(up=W.bfloat16()), "up_weight"),
    (dict(gate=W.half()), "gate_weight"),
    (dict(up=torch.zeros(6, 10, device="meta")), "up_weight"),
    (dict(x=torch.zeros(2, 1, device="meta"), gate=torch.zeros((1 << 20) + 1, 1, device="meta"),
          up=torch.zeros((1 << 20) + 1, 1, device="meta")), "1048576"),
])
def test_refusals(kwargs, text) -> None:
    args = {"x": X, "gate": W, "up": W, **kwargs}
    with pytest.raises(ValueError, match=text):
        gated_linear_hip(*args.values())


def test_the_cpu_has_no_kernel() -> None:
    ops = torch.ops.omniwave_amd
    for call in (lambda: gated_linear_hip(X, W, W), lambda: ops.gated_linear_fwd(X, W, W, True),
                 lambda: ops.gated_linear_bwd(torch.zeros(2, 3, 6), NONE, X, W, W, [True] * 3)):
        with pytest.raises(RuntimeError, match="not supported"):
            call()


@pytest.fixture
def launches(monkeypatch):
    calls = []
    monkeypatch.setattr(gated, "_on", lambda *args: calls.append(args))
    monkeypatch.setattr(gated, "gpu_reason", lambda t: None)

    class Anywhere:
        def __init__(self, device):
            pass

        def __enter__(self):
            pass

        def __exit__(self, *args):
            pass

    monkeypatch.setattr(torch.cuda, "device", Anywhere)
    return calls


@pytest.mark.parametrize("bad", [dict(x=X[..., :9]), dict(x=X.double()), dict(gate=W[:5]), dict(up=W.half()),
                                 dict(up=torch.zeros(6, 10, device="meta"))])
def test_what_the_operators_get(launches, bad) -> None:
    t = {"x": X, "gate": W, "up": W, **bad}
    with pytest.raises(ValueError):
        gated._run_forward(*t.values(), True)
    with pytest.raises(ValueError):
        gated._run_backward(torch.zeros(2, 3, 6), NONE, *t.values(), [True] * 3)
    assert not launches


@pytest.mark.parametrize("up", [torch.zeros(2, 3, 5), torch.zeros(6, 6), torch.zeros(2, 3, 6).half(), torch.zeros(2, 3, 6, device="meta")])
def test_upstream_gradients(launches, up) -> None:
    with pytest.raises(ValueError, match="upstream"):
        gated._run_backward(up, NONE, X, W, W, [True] * 3)
    assert not launches
    gated._run_backward(torch.zeros(2, 3, 6), NONE, X, W, W, [True] * 3)
    gated._run_backward(torch.zeros(2, 3, 6), NONE, X, W, W, [False] * 3)  # nothing is asked for
    gated._run_forward(X, W, W, False)
    assert len(launches) == 2


def test_kept_products(launches) -> None:
    """Two values of fp32 for each of the result, for many channels; the backward looks at them."""
    sizes = [(rows, c, h) for rows in (0, 1, 64, 65, 128, 129, 192, 300, 5000) for c in (0, 127, 128, 1024, 1025, 1535, 1536, 2048, 2049)
             for h in (6, 16, 1000, 4096)]
    for dtype, code in ((torch.bfloat16, 1), (torch.float16, 2), (torch.float32, 0)):
        for rows, c, h in sizes:
            d = _native.OwGatedLinear(rows=rows, channels=c, hidden=h, dtype=code)
            n = gated._kept_values(torch.zeros(rows, c, dtype=dtype, device="meta"), torch.zeros(h, c, dtype=dtype, device="meta"))
            assert _native.lib().ow_gated_linear_kept(ctypes.byref(d)) == 4 * n and n in (0, 2 * rows * h)
            assert n == (2 * rows * h if c >= (128 if code == 0 else 1536) else 0)
    x, w = torch.zeros(200, 2049), torch.zeros(6, 2049)
    assert gated._run_forward(x, w, w, True)[1].numel() == 2400 and not gated._run_forward(x, w, w, False)[1].numel()
    launches.clear()
    up = torch.zeros(200, 6)
    for kept in (torch.zeros(2399), torch.zeros(2400).half(), torch.zeros(2400, device="meta")):
        with pytest.raises(ValueError, match="kept"):
            gated._run_backward(up, kept, x, w, w, [True] * 3)
    assert not launches
    for kept in (torch.zeros(2400), NONE):
        gated._run_backward(up, kept, x, w, w, [True] * 3)
    assert len(launches) == 2


def test_c_entry_points_check_their_arguments() -> None:
    lib, p = _native.lib(), ctypes.c_void_p(256)

    def desc(**kw):
        d = _native.OwGatedLinear(rows=100, x_stride=10, x=256, gate_weight=256, up_weight=256, channels=10, hidden=6, dtype=1)
        for k, v in kw.items():
            setattr(d, k, v)
        return ctypes.byref(d)

    def refused(rc, text, code=1):
        assert rc == code and text in lib.ow_last_error(), lib.ow_last_error()

    refused(lib.ow_gated_linear_fwd(None, p, None, None, 0, None), b"NULL")
    refused(lib.ow_gated_linear_fwd(desc(dtype=3), p, None, None, 0, None), b"dtype", 2)
    refused(lib.ow_gated_linear_fwd(desc(hidden=-1), p, None, None, 0, None), b"negative")
    refused(lib.ow_gated_linear_fwd(desc(channels=(1 << 20) + 1), p, None, None, 0, None), b"at most", 2)
    refused(lib.ow_gated_linear_fwd(desc(rows=1 << 31), p, None, None, 0, None), b"2^31", 2)
    refused(lib.ow_gated_linear_fwd(desc(up_weight=None), p, None, None, 0, None), b"NULL")
    refused(lib.ow_gated_linear_fwd(desc(x=257), p, None, None, 0, None), b"aligned")
    refused(lib.ow_gated_linear_fwd(desc(), None, None, None, 0, None), b"NULL")
    refused(lib.ow_gated_linear_fwd(desc(channels=0), p, None, None, 0, None), b"no channels")
    assert lib.ow_gated_linear_fwd(desc(rows=0), None, None, None, 0, None) == 0 and lib.ow_gated_linear_fwd(desc(hidden=0), None, None, None, 0, None) == 0
    assert lib.ow_gated_linear_bwd_workspace(None) == 0 and lib.ow_gated_linear_bwd_workspace(desc(rows=0)) == 0
    need = lib.ow_gated_linear_bwd_workspace(desc())
    assert need >= 2 * 100 * 6 * 2

    def bwd(d, dh=p, ws=p, n=need, kept=None):
        return lib.ow_gated_linear_bwd(d, kept, dh, 6, p, p, p, ws, n, None)

    for empty in (dict(rows=0), dict(channels=0), dict(hidden=0)):
        refused(bwd(desc(**empty)), b"empty")
    refused(bwd(desc(), dh=None), b"NULL")
    refused(bwd(desc(), dh=ctypes.c_void_p(257)), b"aligned")
    refused(bwd(desc(), kept=ctypes.c_void_p(258)), b"aligned")
    # rows of 10 values fill no whole pieces: x and the weights are copied
    many = desc(rows=20000)
    space = lib.ow_gated_linear_fwd_workspace(many)
    assert space >= (20000 + 2 * 6) * 32 and lib.ow_gated_linear_fwd_workspace(None) == 0
    assert lib.ow_gated_linear_fwd_workspace(desc(rows=64)) == 0
    assert lib.ow_gated_linear_fwd_workspace(desc(rows=20000, channels=8, x_stride=8)) == 0
    refused(lib.ow_gated_linear_fwd(many, p, None, None, 0, None), b"workspace")
    refused(lib.ow_gated_linear_fwd(many, p, None, p, space - 1, None), b"workspace")
    refused(lib.ow_gated_linear_fwd(many, p, None, ctypes.c_void_p(264), space, None), b"workspace")
    refused(lib.ow_gated_linear_fwd(many, p, p, p, space, None), b"kept")
    refused(bwd(many, kept=p), b"kept")
    refused(lib.ow_gated_linear_fwd(desc(channels=1536), p, ctypes.c_void_p(258), None, 0, None), b"kept")
    assert lib.ow_gated_linear_kept(None) == 0 and lib.ow_gated_linear_kept(desc(channels=1536)) == 2 * 100 * 6 * 4
    refused(bwd(desc(), ws=None), b"workspace")
    refused(bwd(desc(), n=need - 1), b"workspace")
    refused(bwd(desc(), ws=ctypes.c_void_p(264)), b"workspace")
