"""The gated feed-forward product with its gradients, as HIP kernels (``gated_linear.hip``, ``gated_linear_bwd.hip``); no
counterpart in the reference, whose gated products stay inside 16 tokens and a channel group.

A plain call is native, its autograd node included (``torch_glue.cpp``); the operator
``omniwave_amd::gated_linear_fwd`` takes the others (compilation, tracing, transforms, tensors to copy first).
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch import Tensor

from omniwave_amd import _native
from omniwave_amd.hip import _DTYPE_CODE, SUPPORTED_DTYPES, _plain
from omniwave_amd.norms import _on, _rows, gpu_reason

MAX_WIDTH = 1 << 20  # channels, hidden


def _ready(x, gate_weight, up_weight) -> None:
    """Raise for what the kernels do not take, before anything touches the GPU, and where they cannot run."""
    if x.dtype not in SUPPORTED_DTYPES:
        raise ValueError(f"unsupported dtype {x.dtype}; expected float16, bfloat16 or float32")
    if x.dim() < 1:
        raise ValueError("x must be [..., C], got a scalar")
    if gate_weight.dim() != 2 or gate_weight.shape[1] != x.shape[-1]:
        raise ValueError(f"gate_weight must be [hidden, {x.shape[-1]}], got {tuple(gate_weight.shape)}")
    if up_weight.shape != gate_weight.shape:
        raise ValueError(f"up_weight must be {tuple(gate_weight.shape)} as gate_weight, got {tuple(up_weight.shape)}")
    for name, w in (("gate_weight", gate_weight), ("up_weight", up_weight)):
        if w.dtype != x.dtype or w.device != x.device:
            raise ValueError(f"{name} must be {x.dtype} on {x.device} as x, got {w.dtype} on {w.device}")
    if max(gate_weight.shape) > MAX_WIDTH:
        raise ValueError(f"weights of {tuple(gate_weight.shape)}; at most {MAX_WIDTH} channels and hidden values are supported")
    if math.prod(x.shape[:-1]) >= 1 << 31:
        raise ValueError(f"{math.prod(x.shape[:-1])} rows; fewer than 2^31 are supported")
    reason = gpu_reason(x)
    if reason is not None:
        raise RuntimeError(f"hip gated linear not supported: {reason}")


def _descriptor(x, gate_weight, up_weight):
    """The C descriptor and the tensors it points into."""
    x, stride = _rows(x)
    keep = [x, gate_weight.contiguous(), up_weight.contiguous()]
    return _native.OwGatedLinear(math.prod(x.shape[:-1]), stride, *[t.data_ptr() for t in keep], x.shape[-1],
                                 gate_weight.shape[0], _DTYPE_CODE[x.dtype]), keep


def _kept_values(x, gate_weight) -> int:
    """Values of both products that a forward keeps for its backward, 0 where that forms them again (the library's
    ``ow_gated_linear_kept``, for sizes that are not yet known, too)."""
    return 2 * math.prod(x.shape[:-1]) * gate_weight.shape[0] if x.shape[-1] >= (128 if x.dtype == torch.float32 else 1536) else 0


def _run_forward(x, gate_weight, up_weight, keep) -> tuple[Tensor, Tensor]:
    """(the result, what the backward needs beside the inputs: both products in float32, or nothing)."""
    _ready(x, gate_weight, up_weight)  # the operator may be called by its name
    h = torch.empty((*x.shape[:-1], gate_weight.shape[0]), dtype=x.dtype, device=x.device)
    kept = torch.empty(_kept_values(x, gate_weight) if keep else 0, dtype=torch.float32, device=x.device)
    if not x.shape[-1]:
        return h.zero_(), kept
    if h.numel():
        desc, _keep = _descriptor(x, gate_weight, up_weight)
        lib = _native.lib()
        with torch.cuda.device(x.device):  # the size goes by the device's compute units
            ws_bytes = lib.ow_gated_linear_fwd_workspace(ctypes.byref(desc))
        workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device) if ws_bytes else None
        _on(x.device, lib.ow_gated_linear_fwd, ctypes.byref(desc), h.data_ptr(), kept.data_ptr() if kept.numel() else None,
            None if workspace is None else workspace.data_ptr(), ws_bytes)
    return h, kept


def _run_backward(dh, kept, x, gate_weight, up_weight, want) -> list[Tensor | None]:
    """Gradients of x, gate_weight and up_weight where ``want`` asks for them."""
    _ready(x, gate_weight, up_weight)  # hooks on saved tensors may hand out others
    if kept.numel() and (kept.device != x.device or kept.dtype != torch.float32
                         or kept.numel() != _kept_values(x, gate_weight)):
        raise ValueError(f"the products kept of {tuple(x.shape)} and {tuple(gate_weight.shape)} on {x.device} are {kept.dtype} "
                         f"{tuple(kept.shape)} on {kept.device}")
    shape = (*x.shape[:-1], gate_weight.shape[0])
    if dh.shape != shape or dh.dtype != x.dtype or dh.device != x.device:
        raise ValueError(f"the upstream gradient of {x.dtype} {shape} on {x.device} is {dh.dtype} {tuple(dh.shape)} on "
                         f"{dh.device}")
    grads = [torch.empty_like(t, memory_format=torch.contiguous_format) if w else None
             for t, w in zip((x, gate_weight, up_weight), want)]
    if not x.numel() or not gate_weight.numel():
        return [None if g is None else g.zero_() for g in grads]
    if any(want):
        desc, _keep = _descriptor(x, gate_weight, up_weight)
        dh, dh_stride = _rows(dh)
        kept = kept.contiguous()
        lib = _native.lib()
        with torch.cuda.device(x.device):  # the size goes by the device's compute units
            ws_bytes = lib.ow_gated_linear_bwd_workspace(ctypes.byref(desc))
        workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device)
        _on(x.device, lib.ow_gated_linear_bwd, ctypes.byref(desc), kept.data_ptr() if kept.numel() else None,
            dh.data_ptr(), dh_stride,
            *[None if g is None else g.data_ptr() for g in grads], workspace.data_ptr(), ws_bytes)
    return grads


@torch.library.custom_op("omniwave_amd::gated_linear_fwd", mutates_args=())
def gated_linear_fwd(x: Tensor, gate_weight: Tensor, up_weight: Tensor, keep: bool) -> tuple[Tensor, Tensor]:
    """(``gated_linear_hip``'s result; what the backward needs beside the inputs where ``keep`` says that there will be
    one, which may be nothing)."""
    return _run_forward(x, gate_weight, up_weight, keep)


@gated_linear_fwd.register_fake
def _gated_linear_fwd_fake(x, gate_weight, up_weight, keep):
    return (x.new_empty((*x.shape[:-1], gate_weight.shape[0])),
            x.new_empty(_kept_values(x, gate_weight) if keep else 0, dtype=torch.float32))


@torch.library.custom_op("omniwave_amd::gated_linear_bwd", mutates_args=())
def gated_linear_bwd(dh: Tensor, kept: Tensor, x: Tensor, gate_weight: Tensor, up_weight: Tensor,
                     want: list[bool]) -> tuple[Tensor, Tensor, Tensor]:
    """Gradients of x, gate_weight and up_weight; empty where ``want`` is false."""
    grads = _run_backward(dh, kept, x, gate_weight, up_weight, want)
    return tuple(x.new_empty(0) if g is None else g for g in grads)


@gated_linear_bwd.register_fake
def _gated_linear_bwd_fake(dh, kept, x, gate_weight, up_weight, want):
    return tuple(t.new_empty(t.shape) if w else x.new_empty(0) for t, w in zip((x, gate_weight, up_weight), want))


def _setup_context(ctx, inputs, output):
    ctx.mark_non_differentiable(output[1])
    ctx.save_for_backward(*inputs[:3], output[1])


def _backward(ctx, dh, _kept):
    x, gate_weight, up_weight, kept = ctx.saved_tensors
    want = list(ctx.needs_input_grad[:3])
    grads = gated_linear_bwd(dh, kept, x, gate_weight, up_weight, want)
    return *[g if w else None for g, w in zip(grads, want)], None


gated_linear_fwd.register_autograd(_backward, setup_context=_setup_context)


def gated_linear_hip(x: Tensor, gate_weight: Tensor, up_weight: Tensor) -> Tensor:
    """``silu(x @ gate_weight.T) * (x @ up_weight.T)``, the first half of a gated feed-forward block in one kernel: ``x``
    ``[..., C]`` (rows at any one distance) and weights ``[hidden, C]``, all of one type (float16, bfloat16 or float32),
    to ``[..., hidden]``.  Products and gate are fp32 and the result is rounded once.  Differentiable once in all three.  The
    backward rounds the gradients of both products to the type in between; where C is large (1,536 for 16-bit types, 128 for
    float32) the forward of a call with a graph keeps both products for it, 8 bytes a value, else they are formed again.

    float32 of many rows (more than 128, and more than fit one round of the kernel for few) runs on the bf16 matrix cores in
    three-part operands: an infinity makes its results NaN, and values below about 2^-110 are held to fewer than 24 bits."""
    glue = _native.glue()
    if glue is not None and _plain(x, gate_weight, up_weight):
        h = glue.gated_linear(x, gate_weight, up_weight)
        if h is not None:
            return h
    # Everything else is checked, and goes through the operator.
    _ready(x, gate_weight, up_weight)
    keep = torch.is_grad_enabled() and any(t.requires_grad for t in (x, gate_weight, up_weight))
    return gated_linear_fwd(x, gate_weight, up_weight, keep)[0]
