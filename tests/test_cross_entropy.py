"""Cross-entropy: what the call refuses, on the CPU, and the C entry points' argument checks."""

from __future__ import annotations

import ctypes

import pytest
import torch

from omniwave_amd import _native, cross_entropy_hip

X, T = torch.zeros(4, 10), torch.zeros(4, dtype=torch.int64)


@pytest.mark.parametrize("kwargs,text", [
    (dict(logits=X.double()), "dtype"),
    (dict(logits=torch.zeros(4, 0)), "classes"),
    (dict(logits=torch.zeros(())), "classes"),
    (dict(target=T.int()), "target"),
    (dict(target=T[:3]), "target"),
    (dict(target=T[:, None]), "target"),
    (dict(target_b=T), "together"),
    (dict(mix=0.5), "together"),
    (dict(target_b=T.float(), mix=0.5), "target_b"),
    (dict(target_b=T, mix=1.5), "mix"),
    (dict(target_b=T, mix=torch.ones(3)), "mix"),
    (dict(target_b=T, mix=torch.ones(4, requires_grad=True)), "no gradient"),
    (dict(label_smoothing=1.1), "label_smoothing"),
    (dict(label_smoothing=float("nan")), "label_smoothing"),
    (dict(reduction="batchmean"), "reduction"),
    (dict(ignore_index=None), "ignore_index"),
])
def test_refusals(kwargs, text) -> None:
    args = dict(logits=X, target=T)
    args.update(kwargs)
    with pytest.raises(ValueError, match=text):
        cross_entropy_hip(args.pop("logits"), args.pop("target"), **args)


def test_the_cpu_has_no_kernel() -> None:
    with pytest.raises(RuntimeError, match="not supported"):
        cross_entropy_hip(X, T)


def test_c_entry_points_check_their_arguments() -> None:
    lib, p = _native.lib(), ctypes.c_void_p(256)

    def desc(**kw):
        d = _native.OwCrossEntropy(rows=4, classes=10, row_stride=10, ignore_index=-100, logits=256, target=256,
                                   smoothing=0.0, dtype=_native.OW_DTYPE_F32, reduction=2)
        for k, v in kw.items():
            setattr(d, k, v)
        return ctypes.byref(d)

    def refused(rc, text, code=1):
        assert rc == code and text in lib.ow_last_error(), lib.ow_last_error()

    def fwd(d, stats=p, losses=p, loss=p, weight=p, ws=None, n=0):
        return lib.ow_cross_entropy_fwd(d, stats, losses, loss, weight, ws, n, None)

    refused(fwd(None), b"NULL")
    refused(fwd(desc(dtype=5)), b"dtype", 2)
    refused(fwd(desc(reduction=3)), b"reduction")
    refused(fwd(desc(rows=-1)), b"rows")
    refused(fwd(desc(classes=0)), b"classes")
    refused(fwd(desc(classes=1 << 30)), b"2^30", 2)
    refused(fwd(desc(rows=1 << 31)), b"2^31", 2)
    refused(fwd(desc(target=None)), b"target")
    refused(fwd(desc(smoothing=2.0)), b"smoothing")
    refused(fwd(desc(), stats=None), b"stats")
    refused(fwd(desc(), weight=None), b"weight")
    refused(fwd(desc(classes=100000)), b"workspace")
    assert fwd(desc(rows=0, reduction=0)) == 0
    assert lib.ow_cross_entropy_workspace(desc()) == 0
    assert lib.ow_cross_entropy_workspace(desc(classes=100000)) >= 4 * 2 * 12
    assert lib.ow_cross_entropy_workspace(None) == 0
    refused(lib.ow_cross_entropy_bwd(desc(), p, p, None, p, None), b"NULL")
    assert lib.ow_cross_entropy_bwd(desc(rows=0), None, None, None, None, None) == 0
