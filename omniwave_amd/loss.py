"""Softmax cross-entropy of logits with its gradient, as HIP kernels (``cross_entropy.hip``).

A plain call is native, its autograd node included (``torch_glue.cpp``); the operator
``omniwave_amd::cross_entropy_fwd`` takes the others (compilation, tracing, transforms, tensors to copy first).
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch import Tensor

from omniwave_amd import _native
from omniwave_amd.hip import _DTYPE_CODE, SUPPORTED_DTYPES, _plain
from omniwave_amd.norms import _on, _rows, gpu_reason


def _check(logits, target, target_b, mix, label_smoothing, ignore_index, reduction) -> None:
    """Raise for what the kernels do not take, before anything touches the GPU."""
    if reduction not in _native.OW_REDUCE:
        raise ValueError(f"reduction must be 'none', 'sum' or 'mean', got {reduction!r}")
    if not isinstance(ignore_index, int):
        raise ValueError(f"ignore_index must be an integer, got {ignore_index!r}")
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError(f"label_smoothing must be in [0, 1], got {label_smoothing}")
    if (target_b is None) != (mix is None):
        raise ValueError("target_b and mix, the weight of target, come together")
    if isinstance(mix, Tensor):
        if mix.requires_grad:
            raise ValueError("mix carries no gradient; detach it")
    elif mix is not None and not 0.0 <= mix <= 1.0:
        raise ValueError(f"mix must be in [0, 1], got {mix}")
    _ready(logits, target, target_b, mix if isinstance(mix, Tensor) else None)


def _ready(logits, target, target_b, mix) -> None:
    """Raise for tensors that the kernels do not take, and where they cannot run."""
    if logits.dtype not in SUPPORTED_DTYPES:
        raise ValueError(f"unsupported dtype {logits.dtype}; expected float16, bfloat16 or float32")
    if logits.dim() < 1 or not 1 <= logits.shape[-1] < 1 << 30:
        raise ValueError(f"logits must be [..., classes] with 1 to 2^30 - 1 classes, got {tuple(logits.shape)}")
    if math.prod(logits.shape[:-1]) >= 1 << 31:
        raise ValueError(f"{math.prod(logits.shape[:-1])} rows; fewer than 2^31 are supported")
    for name, t in (("target", target), ("target_b", target_b)):
        if t is not None and (t.dtype != torch.int64 or t.shape != logits.shape[:-1] or t.device != logits.device):
            raise ValueError(f"{name} must be int64 {tuple(logits.shape[:-1])} on {logits.device}, got {t.dtype} "
                             f"{tuple(t.shape)} on {t.device}")
    if mix is not None and (mix.shape != target.shape or not mix.is_floating_point() or mix.device != logits.device):
        raise ValueError(f"mix must be a number or floating point {tuple(target.shape)} on {logits.device}, got "
                         f"{mix.dtype} {tuple(mix.shape)} on {mix.device}")
    reason = gpu_reason(logits)
    if reason is not None:
        raise RuntimeError(f"hip cross-entropy not supported: {reason}")


def _descriptor(logits, target, target_b, mix, mix_value, label_smoothing, ignore_index, reduction):
    """The C descriptor and the tensors it points into."""
    logits, stride = _rows(logits)
    keep = [logits, *[None if t is None else t.contiguous() for t in (target, target_b)],
            None if mix is None else mix.to(torch.float32).contiguous()]
    return _native.OwCrossEntropy(target.numel(), logits.shape[-1], stride, ignore_index,
                                  *[None if t is None else t.data_ptr() for t in keep], mix_value, label_smoothing,
                                  _DTYPE_CODE[logits.dtype], reduction), keep


def _run_forward(logits, target, target_b, mix, mix_value, label_smoothing, ignore_index,
                 reduction) -> tuple[Tensor, Tensor]:
    """(the loss, or the losses of the rows; what the backward needs beside the inputs: the statistics of the
    rows, a row's weight in the loss and, with a reduction, the losses)."""
    _ready(logits, target, target_b, mix)  # the operator may be called by its name
    device, reduced = logits.device, reduction != 0
    desc, _keep = _descriptor(logits, target, target_b, mix, mix_value, label_smoothing, ignore_index, reduction)
    rows, lib = desc.rows, _native.lib()
    with torch.cuda.device(device):  # the size goes by the device's compute units
        ws_bytes = lib.ow_cross_entropy_workspace(ctypes.byref(desc))
    aux = torch.empty(2 * rows + 1 + (rows if reduced else 0), dtype=torch.float32, device=device)
    loss = torch.empty(() if reduced else target.shape, dtype=torch.float32, device=device)
    workspace = torch.empty(ws_bytes // 4, dtype=torch.float32, device=device) if ws_bytes else None
    at, out = aux.data_ptr(), loss.data_ptr()
    weight = at + 8 * rows
    _on(device, lib.ow_cross_entropy_fwd, ctypes.byref(desc), at, weight + 4 if reduced else out, out if reduced else None,
        weight if reduced else None, None if workspace is None else workspace.data_ptr(), ws_bytes)
    return loss, aux


def _run_backward(up, aux, logits, target, target_b, mix, *options) -> Tensor:
    """The logits' gradient; ``up``: the upstream gradient of the loss (a value) or the losses."""
    _ready(logits, target, target_b, mix)  # hooks on saved tensors may hand out others
    rows, reduced = target.numel(), options[-1] != 0
    if (up.device != logits.device or up.numel() != (1 if reduced else rows) or aux.device != logits.device
            or aux.dtype != torch.float32 or aux.numel() != 2 * rows + 1 + (rows if reduced else 0)):
        raise ValueError(f"the backward of {rows} rows got a gradient of {tuple(up.shape)} on {up.device} and statistics "
                         f"of {aux.dtype} {tuple(aux.shape)} on {aux.device}")
    grad = torch.empty_like(logits, memory_format=torch.contiguous_format)
    if not grad.numel():
        return grad
    desc, _keep = _descriptor(logits, target, target_b, mix, *options)
    up, aux = up.to(torch.float32).contiguous(), aux.contiguous()
    at = aux.data_ptr()
    _on(logits.device, _native.lib().ow_cross_entropy_bwd, ctypes.byref(desc), at,
        at + 8 * desc.rows if desc.reduction else None, up.data_ptr(), grad.data_ptr())
    return grad


_NO_GRADS = (None,) * 7  # of the arguments after the logits


@torch.library.custom_op("omniwave_amd::cross_entropy_fwd", mutates_args=())
def cross_entropy_fwd(logits: Tensor, target: Tensor, target_b: Tensor | None, mix: Tensor | None, mix_value: float,
                      label_smoothing: float, ignore_index: int, reduction: int) -> tuple[Tensor, Tensor]:
    """(the loss, or the losses of the rows; what the backward needs) of ``cross_entropy_hip``."""
    return _run_forward(logits, target, target_b, mix, mix_value, label_smoothing, ignore_index, reduction)


@cross_entropy_fwd.register_fake
def _cross_entropy_fwd_fake(logits, target, target_b, mix, mix_value, label_smoothing, ignore_index, reduction):
    rows = target.numel()
    return (logits.new_empty(() if reduction else target.shape, dtype=torch.float32),
            logits.new_empty(2 * rows + 1 + (rows if reduction else 0), dtype=torch.float32))


@torch.library.custom_op("omniwave_amd::cross_entropy_bwd", mutates_args=())
def cross_entropy_bwd(up: Tensor, aux: Tensor, logits: Tensor, target: Tensor, target_b: Tensor | None,
                      mix: Tensor | None, mix_value: float, label_smoothing: float, ignore_index: int,
                      reduction: int) -> Tensor:
    """The logits' gradient."""
    return _run_backward(up, aux, logits, target, target_b, mix, mix_value, label_smoothing, ignore_index, reduction)


@cross_entropy_bwd.register_fake
def _cross_entropy_bwd_fake(up, aux, logits, target, target_b, mix, mix_value, label_smoothing, ignore_index, reduction):
    return logits.new_empty(logits.shape)


def _setup_context(ctx, inputs, output):
    logits, target, target_b, mix, *options = inputs
    ctx.mark_non_differentiable(output[1])
    ctx.save_for_backward(logits, target, target_b, mix, output[1])
    ctx.options = options


def _backward(ctx, up, _aux):
    logits, target, target_b, mix, aux = ctx.saved_tensors
    return cross_entropy_bwd(up, aux, logits, target, target_b, mix, *ctx.options), *_NO_GRADS


cross_entropy_fwd.register_autograd(_backward, setup_context=_setup_context)


def cross_entropy_hip(logits: Tensor, target: Tensor, *, target_b: Tensor | None = None,
                      mix: Tensor | float | None = None, label_smoothing: float = 0.0, ignore_index: int = -100,
                      reduction: str = "mean") -> Tensor:
    """Cross-entropy of ``softmax(logits)`` (``[..., classes]``, float16, bfloat16 or float32, rows at any
    one distance) and int64 labels ``target`` (``[...]``), as ``torch.nn.functional.cross_entropy`` has it
    for class labels, in float32 whatever the logits' dtype.

    ``target_b`` with ``mix``: a second label of weight ``1 - mix`` beside the first one's ``mix`` (mixed
    images; a number or one for each row).  ``label_smoothing``: the weight of the uniform distribution.
    Rows whose ``target`` is ``ignore_index`` count neither in the loss nor in the mean, and have no
    gradient; a mean of no rows is NaN.  A label outside ``[0, classes)`` makes its row NaN (in ``target_b``, of a
    weight above 0, ``ignore_index`` too), and so does a NaN logit.
    ``reduction``: ``"mean"``, ``"sum"`` or ``"none"``.  Differentiable once in the logits.
    """
    glue, code = _native.glue(), _native.OW_REDUCE.get(reduction)
    number = mix is None or not isinstance(mix, Tensor)  # mix for all rows, or none
    if glue is not None and code is not None and (target_b is None) == (mix is None) \
            and _plain(logits, target, target_b, None if number else mix):
        loss = glue.cross_entropy(logits, target, target_b, None if number else mix, 1.0 if mix is None or not number else mix,
                                  label_smoothing, ignore_index, code)
        if loss is not None:
            return loss
    # Everything else is checked, and goes through the operator.
    _check(logits, target, target_b, mix, label_smoothing, ignore_index, reduction)
    return cross_entropy_fwd(logits, target, target_b, None if number else mix, 1.0 if mix is None or not number else float(mix),
                             float(label_smoothing), ignore_index, code)[0]
