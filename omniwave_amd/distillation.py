"""Distillation of logits from a teacher's top logits with its gradient, as HIP kernels (``distillation.hip``); no
counterpart in the reference.

A plain call is native, its autograd node included (``torch_glue.cpp``); the operator
``omniwave_amd::distillation_fwd`` takes the others (compilation, tracing, transforms, tensors to copy first).
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch import Tensor

from omniwave_amd import _native
from omniwave_amd.hip import _DTYPE_CODE, SUPPORTED_DTYPES, _plain
from omniwave_amd.norms import _on, _rows, gpu_reason

MAX_ENTRIES = 1 << 16  # of a row


def _check(logits, teacher_logits, teacher_indices, temperature, ignore_index, reduction) -> None:
    """Raise for what the kernels do not take, before anything touches the GPU."""
    if reduction not in _native.OW_REDUCE:
        raise ValueError(f"reduction must be 'none', 'sum' or 'mean', got {reduction!r}")
    if not isinstance(ignore_index, int):
        raise ValueError(f"ignore_index must be an integer, got {ignore_index!r}")
    if teacher_logits.requires_grad:
        raise ValueError("teacher_logits carry no gradient; detach them")
    _ready(logits, teacher_logits, teacher_indices, temperature)


def _ready(logits, teacher_logits, teacher_indices, temperature) -> None:
    """Raise for tensors that the kernels do not take, and where they cannot run."""
    if logits.dtype not in SUPPORTED_DTYPES:
        raise ValueError(f"unsupported dtype {logits.dtype}; expected float16, bfloat16 or float32")
    if logits.dim() < 1 or not 1 <= logits.shape[-1] < 1 << 30:
        raise ValueError(f"logits must be [..., classes] with 1 to 2^30 - 1 classes, got {tuple(logits.shape)}")
    if math.prod(logits.shape[:-1]) >= 1 << 31:
        raise ValueError(f"{math.prod(logits.shape[:-1])} rows; fewer than 2^31 are supported")
    want = (*logits.shape[:-1], teacher_logits.shape[-1] if teacher_logits.dim() else 0)
    if teacher_logits.shape != want or teacher_logits.dtype not in SUPPORTED_DTYPES or teacher_logits.device != logits.device:
        raise ValueError(f"teacher_logits must be float16, bfloat16 or float32 {(*logits.shape[:-1], 'entries')} on "
                         f"{logits.device}, got {teacher_logits.dtype} {tuple(teacher_logits.shape)} on {teacher_logits.device}")
    if want[-1] > MAX_ENTRIES:
        raise ValueError(f"{want[-1]} entries a row; at most {MAX_ENTRIES} are supported")
    if teacher_indices.dtype != torch.int64 or teacher_indices.shape != want or teacher_indices.device != logits.device:
        raise ValueError(f"teacher_indices must be int64 {want} on {logits.device}, got {teacher_indices.dtype} "
                         f"{tuple(teacher_indices.shape)} on {teacher_indices.device}")
    # The kernels hold it in float32, and its square.
    if not 1e-15 <= temperature <= 1e15:
        raise ValueError(f"temperature must be in [1e-15, 1e15], got {temperature}")
    reason = gpu_reason(logits)
    if reason is not None:
        raise RuntimeError(f"hip distillation not supported: {reason}")


def _descriptor(logits, teacher_logits, teacher_indices, temperature, ignore_index, reduction):
    """The C descriptor and the tensors it points into."""
    logits, stride = _rows(logits)
    keep = [logits, teacher_logits.contiguous(), teacher_indices.contiguous()]
    return _native.OwDistillation(math.prod(logits.shape[:-1]), logits.shape[-1], stride, ignore_index,
                                  *[t.data_ptr() for t in keep], teacher_logits.shape[-1], _DTYPE_CODE[logits.dtype],
                                  _DTYPE_CODE[teacher_logits.dtype], reduction, temperature), keep


def _run_forward(logits, teacher_logits, teacher_indices, temperature, ignore_index, reduction) -> tuple[Tensor, Tensor]:
    """(the loss, or the losses of the rows; what the backward needs beside the inputs: the statistics of the
    rows, a row's weight in the loss and, with a reduction, the losses)."""
    _ready(logits, teacher_logits, teacher_indices, temperature)  # the operator may be called by its name
    device, reduced = logits.device, reduction != 0
    desc, _keep = _descriptor(logits, teacher_logits, teacher_indices, temperature, ignore_index, reduction)
    rows, lib = desc.rows, _native.lib()
    with torch.cuda.device(device):  # the size goes by the device's compute units
        ws_bytes = lib.ow_distillation_workspace(ctypes.byref(desc))
    aux = torch.empty(4 * rows + 1 + (rows if reduced else 0), dtype=torch.float32, device=device)
    loss = torch.empty(() if reduced else logits.shape[:-1], dtype=torch.float32, device=device)
    workspace = torch.empty(ws_bytes // 4, dtype=torch.float32, device=device) if ws_bytes else None
    at, out = aux.data_ptr(), loss.data_ptr()
    weight = at + 16 * rows
    _on(device, lib.ow_distillation_fwd, ctypes.byref(desc), at, weight + 4 if reduced else out, out if reduced else None,
        weight if reduced else None, None if workspace is None else workspace.data_ptr(), ws_bytes)
    return loss, aux


def _run_backward(up, aux, logits, teacher_logits, teacher_indices, temperature, ignore_index, reduction) -> Tensor:
    """The logits' gradient; ``up``: the upstream gradient of the loss (a value) or the losses."""
    _ready(logits, teacher_logits, teacher_indices, temperature)  # hooks on saved tensors may hand out others
    rows, reduced = math.prod(logits.shape[:-1]), reduction != 0
    if (up.device != logits.device or up.numel() != (1 if reduced else rows) or aux.device != logits.device
            or aux.dtype != torch.float32 or aux.numel() != 4 * rows + 1 + (rows if reduced else 0)):
        raise ValueError(f"the backward of {rows} rows got a gradient of {tuple(up.shape)} on {up.device} and statistics "
                         f"of {aux.dtype} {tuple(aux.shape)} on {aux.device}")
    grad = torch.empty_like(logits, memory_format=torch.contiguous_format)
    if not grad.numel():
        return grad
    desc, _keep = _descriptor(logits, teacher_logits, teacher_indices, temperature, ignore_index, reduction)
    up, aux = up.to(torch.float32).contiguous(), aux.contiguous()
    at = aux.data_ptr()
    _on(logits.device, _native.lib().ow_distillation_bwd, ctypes.byref(desc), at, at + 16 * rows if reduced else None,
        up.data_ptr(), grad.data_ptr())
    return grad


@torch.library.custom_op("omniwave_amd::distillation_fwd", mutates_args=())
def distillation_fwd(logits: Tensor, teacher_logits: Tensor, teacher_indices: Tensor, temperature: float,
                     ignore_index: int, reduction: int) -> tuple[Tensor, Tensor]:
    """(the loss, or the losses of the rows; what the backward needs) of ``distillation_hip``."""
    return _run_forward(logits, teacher_logits, teacher_indices, temperature, ignore_index, reduction)


@distillation_fwd.register_fake
def _distillation_fwd_fake(logits, teacher_logits, teacher_indices, temperature, ignore_index, reduction):
    rows = math.prod(logits.shape[:-1])
    return (logits.new_empty(() if reduction else logits.shape[:-1], dtype=torch.float32),
            logits.new_empty(4 * rows + 1 + (rows if reduction else 0), dtype=torch.float32))


@torch.library.custom_op("omniwave_amd::distillation_bwd", mutates_args=())
def distillation_bwd(up: Tensor, aux: Tensor, logits: Tensor, teacher_logits: Tensor, teacher_indices: Tensor,
                     temperature: float, ignore_index: int, reduction: int) -> Tensor:
    """The logits' gradient."""
    return _run_backward(up, aux, logits, teacher_logits, teacher_indices, temperature, ignore_index, reduction)


@distillation_bwd.register_fake
def _distillation_bwd_fake(up, aux, logits, teacher_logits, teacher_indices, temperature, ignore_index, reduction):
    return logits.new_empty(logits.shape)


def _setup_context(ctx, inputs, output):
    logits, teacher_logits, teacher_indices, *options = inputs
    ctx.mark_non_differentiable(output[1])
    ctx.save_for_backward(logits, teacher_logits, teacher_indices, output[1])
    ctx.options = options


def _backward(ctx, up, _aux):
    logits, teacher_logits, teacher_indices, aux = ctx.saved_tensors
    return distillation_bwd(up, aux, logits, teacher_logits, teacher_indices, *ctx.options), None, None, None, None, None


distillation_fwd.register_autograd(_backward, setup_context=_setup_context)


def distillation_hip(logits: Tensor, teacher_logits: Tensor, teacher_indices: Tensor, *, temperature: float = 1.0,
                     ignore_index: int = -100, reduction: str = "mean") -> Tensor:
    """Loss of ``logits`` (``[..., classes]``, float16, bfloat16 or float32, rows at any one distance) against a
    teacher's top logits: ``teacher_logits`` (``[..., entries]``, any of these types) of the classes
    ``teacher_indices`` (int64, the same shape).  With ``T = temperature`` and ``q = softmax(teacher_logits / T)`` over
    a row's entries, a row's loss is ``T^2 * sum_j q_j (ln q_j - ln softmax(logits / T)[index_j])``, the divergence of the
    student's distribution from the teacher's; ``T^2`` keeps the gradient's scale.  In float32 whatever the logits'
    dtype.

    Entries whose index is ``ignore_index``, or whose logit is -inf, are none (lists of several lengths); rows without an
    entry count neither in the loss nor in the mean, and have no gradient; a mean of no rows is NaN.  A class may have
    several entries.  An index outside ``[0, classes)``, or a NaN logit, makes its row NaN.
    ``reduction``: ``"mean"``, ``"sum"`` or ``"none"``.  Differentiable once in the logits.

    A row whose entries are all classes, one each, has a loss with the digits of fp32 however small it is; that of a shorter list,
    which is at least the share of the classes left out, is off by a few 1e-7 of ``T^2`` besides.
    """
    glue, code = _native.glue(), _native.OW_REDUCE.get(reduction)
    if glue is not None and code is not None and _plain(logits, teacher_logits, teacher_indices):
        loss = glue.distillation(logits, teacher_logits, teacher_indices, temperature, ignore_index, code)
        if loss is not None:
            return loss
    # Everything else is checked, and goes through the operator.
    _check(logits, teacher_logits, teacher_indices, temperature, ignore_index, reduction)
    return distillation_fwd(logits, teacher_logits, teacher_indices, float(temperature), ignore_index, code)[0]
