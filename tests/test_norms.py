"""Norms around a block: what the calls refuse, on the CPU, and the C entry points' argument checks."""

from __future__ import annotations

import ctypes

import pytest
import torch

from omniwave_amd import _native, block_norms_hip, rms_norm_hip
from omniwave_amd.norms import _check, _rows

X = torch.zeros(2, 3, 8)
W = torch.ones(8)


@pytest.mark.parametrize("kwargs,text", [
    (dict(x=X.double()), "dtype"),
    (dict(x=X.int()), "dtype"),
    (dict(x=torch.zeros(8)), r"\[B, ..., C\]"),
    (dict(x=torch.zeros(2, 8193), delta=torch.zeros(2, 8193)), "channels"),
    (dict(delta=torch.zeros(2, 8)), "delta"),
    (dict(delta=X.bfloat16()), "delta"),
    (dict(post_weight=torch.ones(7)), "post_weight"),
    (dict(post_weight=torch.ones(2, 8)), "post_weight"),
    (dict(next_weight=torch.ones(1)), "next_weight"),
    (dict(next_weight=W.double()), "next_weight"),
    (dict(gate=torch.ones(3, 8)), "gate"),
    (dict(gate=torch.ones(2, 1, 8)), "gate"),
    (dict(scale=torch.ones(3)), "scale"),
    (dict(scale=torch.ones(2, dtype=torch.int32)), "scale"),
    (dict(scale=torch.ones(2, requires_grad=True)), "no gradient"),
    (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"),
])
def test_refusals(kwargs, text) -> None:
    args = dict(x=X, delta=X if "x" not in kwargs else kwargs["x"])
    args.update(kwargs)
    x, delta = args.pop("x"), args.pop("delta")
    with pytest.raises(ValueError, match=text):
        block_norms_hip(x, delta, **args)


def test_missing_inputs() -> None:
    with pytest.raises(ValueError, match="delta"):
        block_norms_hip(X, None)
    with pytest.raises(ValueError, match="weight"):
        rms_norm_hip(X, None)


def test_the_cpu_has_no_kernel() -> None:
    with pytest.raises(RuntimeError, match="not supported"):
        rms_norm_hip(X, W)


def test_a_gate_of_one_image_is_told_by_its_dimensions() -> None:
    x = torch.zeros(8, 8)
    _check(x, x, None, torch.ones(8), None, None, 1e-6)
    _check(x, x, None, torch.ones(8, 8), None, None, 1e-6)


@pytest.mark.parametrize("t,step", [
    (torch.zeros(2, 3, 16)[..., :8], 16),
    (torch.zeros(2, 3, 16)[..., 1:9], 16),
    (torch.zeros(8).expand(2, 3, 8), 0),
    (torch.zeros(4, 3, 8)[::2], 8),            # images apart: copied
    (torch.zeros(2, 8, 3).transpose(1, 2), 8),  # values apart: copied
    (torch.zeros(1, 1, 8), 8),
    (torch.zeros(6, 2, 8)[:, :1], 16),
    (torch.zeros(5, 2)[:, :1], 2),
])
def test_rows(t, step) -> None:
    r, got = _rows(t)
    assert got == step and torch.equal(r, t)
    if r.data_ptr() == t.data_ptr() and r.is_contiguous() == t.is_contiguous():
        flat = t.reshape(-1, t.shape[-1])
        assert all(r.storage_offset() + i * step < r.untyped_storage().nbytes() // r.element_size()
                   for i in range(flat.shape[0]))


def test_c_entry_points_check_their_arguments() -> None:
    lib, p = _native.lib(), ctypes.c_void_p(256)
    f32 = _native.OW_DTYPE_F32

    def desc(**kw):
        d = _native.OwBlockNorms(rows=6, rows_per_image=3, x_stride=8, delta_stride=8, x=256, delta=256, channels=8,
                                 dtype=f32, eps=1e-6)
        for k, v in kw.items():
            setattr(d, k, v)
        return ctypes.byref(d)

    def refused(rc, text, code=1):
        assert rc == code and text in lib.ow_last_error()

    refused(lib.ow_block_norms_fwd(None, p, None, None), b"NULL")
    refused(lib.ow_block_norms_fwd(desc(dtype=7), p, None, None), b"dtype", 2)
    refused(lib.ow_block_norms_fwd(desc(rows=-1), p, None, None), b"negative")
    refused(lib.ow_block_norms_fwd(desc(channels=8193), p, None, None), b"channels", 2)
    refused(lib.ow_block_norms_fwd(desc(rows=1 << 31, rows_per_image=1 << 31), p, None, None), b"rows", 2)
    refused(lib.ow_block_norms_fwd(desc(rows_per_image=4), p, None, None), b"whole images")
    refused(lib.ow_block_norms_fwd(desc(x=None), p, None, None), b"x is NULL")
    refused(lib.ow_block_norms_fwd(desc(delta=None, gate=256), None, p, None), b"need delta")
    refused(lib.ow_block_norms_fwd(desc(gate=256, gate_dtype=9), p, None, None), b"weight dtype")
    refused(lib.ow_block_norms_fwd(desc(), None, None, None), b"out is written")
    refused(lib.ow_block_norms_fwd(desc(next_weight=256), p, None, None), b"next is written")
    refused(lib.ow_block_norms_fwd(desc(delta=None), None, None, None), b"neither")
    assert lib.ow_block_norms_fwd(desc(rows=0), p, None, None) == 0
    assert lib.ow_block_norms_bwd_workspace(None) == 0
    many = dict(rows=6000, rows_per_image=3000)
    assert lib.ow_block_norms_bwd_workspace(desc()) == 0  # few rows: one workgroup
    assert lib.ow_block_norms_bwd_workspace(desc(**many)) >= 3 * 8 * 4

    def bwd(d, dout=p, dnext=None, dx=p, ddelta=None, dpost=None, dgate=None, dnw=None, ws=None, n=0):
        return lib.ow_block_norms_bwd(d, dout, 8, dnext, 8, dx, ddelta, dpost, dgate, dnw, ws, n, None)

    refused(bwd(desc(rows=0)), b"no rows")
    refused(bwd(desc(), dnext=p), b"next_weight")
    refused(bwd(desc(), dout=None), b"no upstream")
    refused(bwd(desc(), dgate=p), b"not given")
    refused(bwd(desc(gate=256, **many), dgate=p), b"workspace")
    refused(bwd(desc(gate=256, **many), dgate=p, ws=p, n=8), b"workspace")
