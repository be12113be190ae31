"""Distillation: what the call and its operators refuse, on the CPU, and the C entry points' argument checks."""

from __future__ import annotations

import ctypes

import pytest
import torch

from omniwave_amd import _native, distillation, distillation_hip

X, V, I = torch.zeros(4, 10), torch.zeros(4, 3), torch.zeros(4, 3, dtype=torch.int64)


@pytest.mark.parametrize("kwargs,text", [
    (dict(logits=X.double()), "dtype"),
    (dict(logits=torch.zeros(4, 0)), "classes"),
    (dict(logits=torch.zeros(())), "classes"),
    (dict(teacher_logits=V.double()), "teacher_logits"),
    (dict(teacher_logits=V[:3]), "teacher_logits"),
    (dict(teacher_logits=V[0]), "teacher_logits"),
    (dict(teacher_logits=torch.zeros(())), "teacher_logits"),
    (dict(teacher_logits=torch.zeros(4, 3, device="meta")), "teacher_logits"),
    (dict(teacher_logits=torch.zeros(4, 3, requires_grad=True)), "no gradient"),
    (dict(teacher_indices=I.int()), "teacher_indices"),
    (dict(teacher_indices=I[:, :2]), "teacher_indices"),
    (dict(teacher_logits=torch.zeros(4, 65537), teacher_indices=torch.zeros(4, 65537, dtype=torch.int64)), "65536"),
    (dict(temperature=0.0), "temperature"),
    (dict(temperature=-1.0), "temperature"),
    (dict(temperature=float("nan")), "temperature"),
    (dict(temperature=float("inf")), "temperature"),
    (dict(reduction="batchmean"), "reduction"),
    (dict(ignore_index=None), "ignore_index"),
    (dict(ignore_index=1.5), "ignore_index"),
])
def test_refusals(kwargs, text) -> None:
    args = {"logits": X, "teacher_logits": V, "teacher_indices": I, **kwargs}
    with pytest.raises(ValueError, match=text):
        distillation_hip(args.pop("logits"), args.pop("teacher_logits"), args.pop("teacher_indices"), **args)


def test_the_cpu_has_no_kernel() -> None:
    ops = torch.ops.omniwave_amd
    for call in (lambda: distillation_hip(X, V, I), lambda: ops.distillation_fwd(X, V, I, 1.0, -100, 2),
                 lambda: ops.distillation_bwd(torch.ones(()), torch.zeros(21), X, V, I, 1.0, -100, 2)):
        with pytest.raises(RuntimeError, match="not supported"):
            call()


@pytest.fixture
def launches(monkeypatch):
    calls = []
    monkeypatch.setattr(distillation, "_on", lambda *args: calls.append(args))
    monkeypatch.setattr(distillation, "gpu_reason", lambda t: None)

    class Anywhere:
        def __init__(self, device):
            pass

        def __enter__(self):
            pass

        def __exit__(self, *args):
            pass

    monkeypatch.setattr(torch.cuda, "device", Anywhere)
    return calls


@pytest.mark.parametrize("bad", [dict(logits=X.double()), dict(logits=X[:3]), dict(teacher=V[:, :2]), dict(indices=I[:3]),
                                 dict(indices=I.int()), dict(indices=torch.zeros(4, 3, dtype=torch.int64, device="meta"))])
def test_what_the_operators_get(launches, bad) -> None:
    t = {"logits": X, "teacher": V, "indices": I, **bad}
    with pytest.raises(ValueError):
        distillation._run_forward(*t.values(), 1.0, -100, 2)
    with pytest.raises(ValueError):
        distillation._run_backward(torch.ones(()), torch.zeros(21), *t.values(), 1.0, -100, 2)
    assert not launches


def test_what_the_backward_gets(launches) -> None:
    for up, aux in ((torch.ones(2), torch.zeros(21)), (torch.ones(()), torch.zeros(20)), (torch.ones(()), torch.zeros(21).half()),
                    (torch.ones((), device="meta"), torch.zeros(21)), (torch.ones(()), torch.zeros(21, device="meta"))):
        with pytest.raises(ValueError, match="backward"):
            distillation._run_backward(up, aux, X, V, I, 1.0, -100, 2)
    with pytest.raises(ValueError, match="backward"):
        distillation._run_backward(torch.ones(()), torch.zeros(17), X, V, I, 1.0, -100, 0)  # a gradient for each row
    assert not launches
    distillation._run_backward(torch.ones(()), torch.zeros(21), X, V, I, 1.0, -100, 2)
    distillation._run_backward(torch.ones(4), torch.zeros(17), X, V, I, 1.0, -100, 0)
    assert len(launches) == 2


def test_c_entry_points_check_their_arguments() -> None:
    lib, p = _native.lib(), ctypes.c_void_p(256)

    def desc(**kw):
        d = _native.OwDistillation(rows=4, classes=10, row_stride=10, ignore_index=-100, logits=256, teacher=256, indices=256,
                                   top=3, dtype=0, teacher_dtype=0, reduction=2, temperature=1.0)
        for k, v in kw.items():
            setattr(d, k, v)
        return ctypes.byref(d)

    def refused(rc, text, code=1):
        assert rc == code and text in lib.ow_last_error(), lib.ow_last_error()

    def fwd(d, stats=p, losses=p, loss=p, weight=p, ws=None, n=0):
        return lib.ow_distillation_fwd(d, stats, losses, loss, weight, ws, n, None)

    refused(fwd(None), b"NULL")
    refused(fwd(desc(dtype=5)), b"dtypes", 2)
    refused(fwd(desc(teacher_dtype=5)), b"dtypes", 2)
    refused(fwd(desc(reduction=3)), b"reduction")
    refused(fwd(desc(rows=-1)), b"rows")
    refused(fwd(desc(classes=0)), b"classes")
    refused(fwd(desc(top=-1)), b"entries")
    refused(fwd(desc(top=65537)), b"2^16", 2)
    refused(fwd(desc(classes=1 << 30)), b"2^30", 2)
    refused(fwd(desc(rows=1 << 31)), b"2^31", 2)
    for t in (0.0, -2.0, float("nan"), float("inf"), 1e-20):
        refused(fwd(desc(temperature=t)), b"temperature")
    refused(fwd(desc(teacher=None)), b"teacher")
    refused(fwd(desc(indices=None)), b"indices")
    refused(fwd(desc(), stats=None), b"stats")
    refused(fwd(desc(), weight=None), b"weight")
    refused(fwd(desc(classes=100000)), b"workspace")
    assert fwd(desc(rows=0, reduction=0)) == 0
    assert lib.ow_distillation_workspace(desc()) == 0
    assert lib.ow_distillation_workspace(desc(classes=100000)) >= 4 * 2 * 12
    assert lib.ow_distillation_workspace(None) == 0
    refused(lib.ow_distillation_bwd(desc(), p, p, None, p, None), b"NULL")
    assert lib.ow_distillation_bwd(desc(rows=0), None, None, None, None, None) == 0
