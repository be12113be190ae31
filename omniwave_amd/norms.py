"""The norms around a block with its gate, residual scale and residual, as HIP kernels.

* ``block_norms_hip`` — what lies between a block's delta and the next block's input:
  ``out = x + scale * gate * norm(delta)`` and ``norm(out)``, each read and written once.
* ``rms_norm_hip`` — the norm before a block alone (``bigemm`` takes pre-normalised activations,
  omniweave/ops/bigemm.py:24-36).
* ``layer_norm_hip`` — layer norm of rows, with weight and bias (no counterpart in the reference).

All are differentiable.  The reference has the norm before the block, the LayerScale gate, the drop-path
scale and the residual as eager steps (omniweave/models/block.py:83-108) and no norm after the block;
``OmniWeaveBlock(post_norm=True)`` is the block that has one.  All sums are fp32 and each output is rounded
once from fp32.

A plain call is native, its autograd node included (``torch_glue.cpp``); the operator
``omniwave_amd::block_norms_fwd`` or ``layer_norm_fwd`` takes the others (compilation, tracing, transforms, tensors to copy first).
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch import Tensor

from omniwave_amd import _native
from omniwave_amd.hip import _DTYPE_CODE, SUPPORTED_DTYPES, _device_arch, _plain, _stream_ptr

MAX_CHANNELS = 8192


def gpu_reason(t: Tensor) -> str | None:
    """Why the kernels cannot run on ``t``'s device, or None."""
    err = _native.load_error()
    if err is not None:
        return f"native library unavailable: {err}"
    if not t.is_cuda:
        return f"the tensor is on {t.device}, not on a GPU"
    arch = _device_arch(t.device.index)
    if not arch.startswith("gfx950"):
        return f"device architecture {arch} is not gfx950"
    return None


def _check(x, delta, post_weight, gate, scale, next_weight, eps) -> None:
    """Raise for what the kernels do not take, before anything touches the GPU."""
    if x.dtype not in SUPPORTED_DTYPES:
        raise ValueError(f"unsupported dtype {x.dtype}; expected float16, bfloat16 or float32")
    if x.dim() < 2:
        raise ValueError(f"x must be [B, ..., C], got shape {tuple(x.shape)}")
    b, c = x.shape[0], x.shape[-1]
    if c > MAX_CHANNELS:
        raise ValueError(f"{c} channels; at most {MAX_CHANNELS} are supported")
    if x.numel() and x.numel() // c >= 1 << 31:
        raise ValueError(f"{x.numel() // c} rows; fewer than 2^31 are supported")
    if not (eps >= 0.0 and math.isfinite(eps)):
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    if delta is not None and (delta.shape != x.shape or delta.dtype != x.dtype or delta.device != x.device):
        raise ValueError(f"delta must be {x.dtype} {tuple(x.shape)} on {x.device}, got {delta.dtype} "
                         f"{tuple(delta.shape)} on {delta.device}")
    for name, w in (("post_weight", post_weight), ("gate", gate), ("next_weight", next_weight)):
        if w is None:
            continue
        if w.shape != (c,) and not (name == "gate" and w.shape == (b, c)):
            raise ValueError(f"{name} must be [{c}]{f' or [{b}, {c}]' if name == 'gate' else ''}, got {tuple(w.shape)}")
        if w.dtype not in SUPPORTED_DTYPES or w.device != x.device:
            raise ValueError(f"{name} must be float16, bfloat16 or float32 on {x.device}, got {w.dtype} on {w.device}")
    if scale is not None:
        if scale.shape != (b,) or scale.device != x.device or not scale.is_floating_point():
            raise ValueError(f"scale must be floating point [{b}] on {x.device}, got {scale.dtype} {tuple(scale.shape)} "
                             f"on {scale.device}")
        if scale.requires_grad:
            raise ValueError("scale carries no gradient (a gate of [B, C] does); detach it")


def _ready(x, delta, post_weight, gate, scale, next_weight, eps) -> None:
    """Raise for what the kernels do not take, and where they cannot run."""
    _check(x, delta, post_weight, gate, scale, next_weight, eps)
    reason = gpu_reason(x)
    if reason is not None:
        raise RuntimeError(f"hip norms not supported: {reason}")


def _rows(t: Tensor) -> tuple[Tensor, int]:
    """``t`` or a contiguous copy, with the distance between its rows (the last dimension) in values:
    rows lie at one distance, one value after the other."""
    c = t.shape[-1]
    if t.is_contiguous():
        return t, c
    if c == 1 or t.stride(-1) == 1:
        step, span = None, 0
        for size, stride in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
            if size == 1:
                continue
            if step is None:
                step, span = stride, stride * size
            elif stride == span:
                span *= size
            else:
                break
        else:
            return t, c if step is None else step
    return t.contiguous(), c


def _descriptor(x, delta, post_weight, gate, scale, next_weight, eps):
    """The C descriptor and the tensors it points into."""
    keep = [x, delta, post_weight, gate, scale, next_weight]
    x, x_stride = _rows(x)
    keep[0] = x
    delta_stride = 0
    if delta is not None:
        keep[1], delta_stride = _rows(delta)
    for i in (2, 3, 5):
        if keep[i] is not None:
            keep[i] = keep[i].contiguous()
    if scale is not None:
        keep[4] = scale.to(torch.float32).contiguous()
    rows = x.numel() // x.shape[-1]
    ptr = [None if t is None else t.data_ptr() for t in keep]
    code = [0 if t is None else _DTYPE_CODE[t.dtype] for t in keep]
    return _native.OwBlockNorms(rows, rows // x.shape[0], x_stride, delta_stride, *ptr, x.shape[-1], code[0], code[2],
                                code[3], code[5], int(gate is not None and gate.dim() == 2), eps), keep


def _on(device: torch.device, fn, *args) -> None:
    """One native call on ``device``'s current stream (the call's last argument)."""
    if device.index != torch._C._cuda_getDevice():
        with torch.cuda.device(device):
            _native.check(fn(*args, _stream_ptr(device)), fn.__name__)
    else:
        _native.check(fn(*args, _stream_ptr(device)), fn.__name__)


def _empty(t: Tensor) -> Tensor:
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _run_forward(x, delta, post_weight, gate, scale, next_weight, eps) -> tuple[Tensor | None, Tensor | None]:
    _ready(x, delta, post_weight, gate, scale, next_weight, eps)  # the operator may be called by its name
    out = _empty(x) if delta is not None else None
    nxt = _empty(x) if next_weight is not None else None
    if x.numel():
        desc, _keep = _descriptor(x, delta, post_weight, gate, scale, next_weight, eps)
        _on(x.device, _native.lib().ow_block_norms_fwd, ctypes.byref(desc), None if out is None else out.data_ptr(),
            None if nxt is None else nxt.data_ptr())
    return out, nxt


def _run_backward(dout, dnext, x, delta, post_weight, gate, scale, next_weight, eps, want) -> list[Tensor | None]:
    """Gradients of x, delta, post_weight, gate and next_weight where ``want`` asks for them and they
    exist; ``dout`` / ``dnext`` None: that output has no upstream gradient."""
    _ready(x, delta, post_weight, gate, scale, next_weight, eps)  # hooks on saved tensors may hand out others
    for g in (dout, dnext):
        if g is not None and (g.shape != x.shape or g.dtype != x.dtype or g.device != x.device):
            raise ValueError(f"the upstream gradient of {x.dtype} {tuple(x.shape)} on {x.device} is {g.dtype} "
                             f"{tuple(g.shape)} on {g.device}")
    grads = [_empty(t) if w and t is not None else None for t, w in zip((x, delta, post_weight, gate, next_weight), want)]
    if x.numel() == 0 or (dout is None and dnext is None):
        return [None if g is None else g.zero_() for g in grads]
    ptr = [None if g is None else g.data_ptr() for g in grads]
    if dnext is None and grads[4] is not None:
        grads[4].zero_()
        ptr[4] = None
    desc, _keep = _descriptor(x, delta, post_weight, gate, scale, next_weight, eps)
    upstream = []
    for g in (dout, dnext):
        upstream.append((None, 0) if g is None else _rows(g))
    args = [v for g, stride in upstream for v in (None if g is None else g.data_ptr(), stride)]
    lib, ws_bytes, workspace = _native.lib(), 0, None
    if any(ptr[2:]):
        with torch.cuda.device(x.device):  # the size goes by the device's compute units
            ws_bytes = lib.ow_block_norms_bwd_workspace(ctypes.byref(desc))
        workspace = torch.empty(ws_bytes // 4, dtype=torch.float32, device=x.device) if ws_bytes else None
    _on(x.device, lib.ow_block_norms_bwd, ctypes.byref(desc), *args, *ptr,
        None if workspace is None else workspace.data_ptr(), ws_bytes)
    return grads


@torch.library.custom_op("omniwave_amd::block_norms_fwd", mutates_args=())
def block_norms_fwd(x: Tensor, delta: Tensor | None, post_weight: Tensor | None, gate: Tensor | None,
                    scale: Tensor | None, next_weight: Tensor | None, eps: float) -> tuple[Tensor, Tensor]:
    """(out, next) of ``block_norms_hip``; empty where there is none (``out`` without ``delta``, ``next``
    without ``next_weight``)."""
    out, nxt = _run_forward(x, delta, post_weight, gate, scale, next_weight, eps)
    return x.new_empty(0) if out is None else out, x.new_empty(0) if nxt is None else nxt


@block_norms_fwd.register_fake
def _block_norms_fwd_fake(x, delta, post_weight, gate, scale, next_weight, eps):
    return (x.new_empty(0) if delta is None else x.new_empty(x.shape),
            x.new_empty(0) if next_weight is None else x.new_empty(x.shape))


@torch.library.custom_op("omniwave_amd::block_norms_bwd", mutates_args=())
def block_norms_bwd(dout: Tensor | None, dnext: Tensor | None, x: Tensor, delta: Tensor | None,
                    post_weight: Tensor | None, gate: Tensor | None, scale: Tensor | None, next_weight: Tensor | None,
                    eps: float, want: list[bool]) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    """Gradients of x, delta, post_weight, gate and next_weight; empty where ``want`` is false."""
    grads = _run_backward(dout, dnext, x, delta, post_weight, gate, scale, next_weight, eps, want)
    return tuple(x.new_empty(0) if g is None else g for g in grads)


@block_norms_bwd.register_fake
def _block_norms_bwd_fake(dout, dnext, x, delta, post_weight, gate, scale, next_weight, eps, want):
    return tuple(x.new_empty(0) if t is None or not w else t.new_empty(t.shape)
                 for t, w in zip((x, delta, post_weight, gate, next_weight), want))


def _norms_setup_context(ctx, inputs, output):
    *tensors, eps = inputs
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(*tensors)
    ctx.eps = float(eps)


def _norms_backward(ctx, dout, dnext):
    saved = ctx.saved_tensors  # asked for once: recomputation and hooks answer once
    x, delta, post_weight, gate, scale, next_weight = saved
    need = [n and t is not None for n, t in zip(ctx.needs_input_grad, saved)]
    want = [need[0], need[1], need[2], need[3], need[5]]
    dout, dnext = (dout if delta is not None else None), (dnext if next_weight is not None else None)
    if dout is None and dnext is None:
        return (None,) * 7
    grads = block_norms_bwd(dout, dnext, x, delta, post_weight, gate, scale, next_weight, ctx.eps, want)
    grads = [g if w else None for g, w in zip(grads, want)]
    return grads[0], grads[1], grads[2], grads[3], None, grads[4], None


block_norms_fwd.register_autograd(_norms_backward, setup_context=_norms_setup_context)


def _norms(x, delta, post_weight, gate, scale, next_weight, eps) -> tuple[Tensor | None, Tensor | None]:
    glue = _native.glue()
    if glue is not None and _plain(x, delta, post_weight, gate, scale, next_weight):
        both = glue.norms(x, delta, post_weight, gate, scale, next_weight, eps)
        if both is not None:
            return both
    # Everything else is checked, and goes through the operator.
    eps = float(eps)
    _ready(x, delta, post_weight, gate, scale, next_weight, eps)
    out, nxt = block_norms_fwd(x, delta, post_weight, gate, scale, next_weight, eps)
    return (None if delta is None else out), (None if next_weight is None else nxt)


def block_norms_hip(x: Tensor, delta: Tensor, *, post_weight: Tensor | None = None, gate: Tensor | None = None,
                    scale: Tensor | None = None, next_weight: Tensor | None = None,
                    eps: float = 1e-6) -> tuple[Tensor, Tensor | None]:
    """``(out, next)`` after a block:

    ``out = x + scale * gate * p``, ``p = delta / sqrt(mean(delta^2) + eps) * post_weight`` (``p = delta``
    without ``post_weight``), and ``next = out / sqrt(mean(out^2) + eps) * next_weight``, the next block's
    pre-normalised input (None without ``next_weight``); means over the last dimension.

    ``x``, ``delta``: ``[B, ..., C]`` in float16, bfloat16 or float32, C up to 8,192, rows at any one
    distance.  ``gate``: ``[C]`` (LayerScale) or ``[B, C]`` (a gate made for each image).  ``scale``:
    ``[B]``, the residual scale of each image (drop-path factors as ``drop_path_scale`` draws them);
    it carries no gradient.  Weights may have another dtype than ``x``.  ``next`` is formed from the
    unrounded ``out``.  Differentiable once in x, delta and the weights.
    """
    if delta is None:
        raise ValueError("block_norms_hip needs delta (rms_norm_hip is the norm alone)")
    return _norms(x, delta, post_weight, gate, scale, next_weight, eps)


def rms_norm_hip(x: Tensor, weight: Tensor, eps: float = 1e-6) -> Tensor:
    """``x / sqrt(mean(x^2) + eps) * weight`` over the last dimension, rounded once from fp32: the norm
    before a block (omniweave/models/block.py:83-85 rounds the mean, its root and the product to x's dtype
    on the way).  Shapes, dtypes and gradients as ``block_norms_hip``."""
    if weight is None:
        raise ValueError("rms_norm_hip needs a weight")
    return _norms(x, None, None, None, None, weight, eps)[1]


# ---------------------------------------------------------------------------------------
# Layer norm


def _layer_norm_ready(x, weight, bias, eps) -> None:
    """Raise for what the kernels do not take, before anything touches the GPU, and where they cannot run."""
    if x.dtype not in SUPPORTED_DTYPES:
        raise ValueError(f"unsupported dtype {x.dtype}; expected float16, bfloat16 or float32")
    if x.dim() < 1:
        raise ValueError("x must be [..., C], got a scalar")
    c = x.shape[-1]
    if c > MAX_CHANNELS:
        raise ValueError(f"{c} channels; at most {MAX_CHANNELS} are supported")
    if x.numel() and x.numel() // c >= 1 << 31:
        raise ValueError(f"{x.numel() // c} rows; fewer than 2^31 are supported")
    if not (eps >= 0.0 and math.isfinite(eps)):
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    for name, w in (("weight", weight), ("bias", bias)):
        if w is not None and (w.shape != (c,) or w.dtype not in SUPPORTED_DTYPES or w.device != x.device):
            raise ValueError(f"{name} must be float16, bfloat16 or float32 [{c}] on {x.device}, got {w.dtype} "
                             f"{tuple(w.shape)} on {w.device}")
    reason = gpu_reason(x)
    if reason is not None:
        raise RuntimeError(f"hip layer norm not supported: {reason}")


def _layer_norm_descriptor(x, weight, bias, eps):
    """The C descriptor and the tensors it points into."""
    x, stride = _rows(x)
    keep = [x, *[None if w is None else w.contiguous() for w in (weight, bias)]]
    code = [0 if t is None else _DTYPE_CODE[t.dtype] for t in keep]
    return _native.OwLayerNorm(x.numel() // x.shape[-1], stride, *[None if t is None else t.data_ptr() for t in keep],
                               x.shape[-1], *code, eps), keep


def _run_layer_norm_forward(x, weight, bias, eps) -> Tensor:
    _layer_norm_ready(x, weight, bias, eps)  # the operator may be called by its name
    y = _empty(x)
    if x.numel():
        desc, _keep = _layer_norm_descriptor(x, weight, bias, eps)
        _on(x.device, _native.lib().ow_layer_norm_fwd, ctypes.byref(desc), y.data_ptr())
    return y


def _run_layer_norm_backward(dy, x, weight, bias, eps, want) -> list[Tensor | None]:
    """Gradients of x, weight and bias where ``want`` asks for them and they exist."""
    _layer_norm_ready(x, weight, bias, eps)  # hooks on saved tensors may hand out others
    if dy.shape != x.shape or dy.dtype != x.dtype or dy.device != x.device:
        raise ValueError(f"the upstream gradient of {x.dtype} {tuple(x.shape)} on {x.device} is {dy.dtype} "
                         f"{tuple(dy.shape)} on {dy.device}")
    grads = [_empty(t) if w and t is not None else None for t, w in zip((x, weight, bias), want)]
    if x.numel() == 0:
        return [None if g is None else g.zero_() for g in grads]
    ptr = [None if g is None else g.data_ptr() for g in grads]
    desc, _keep = _layer_norm_descriptor(x, weight, bias, eps)
    dy, dy_stride = _rows(dy)
    lib, ws_bytes, workspace = _native.lib(), 0, None
    if any(ptr[1:]):
        with torch.cuda.device(x.device):  # the size goes by the device's compute units
            ws_bytes = lib.ow_layer_norm_bwd_workspace(ctypes.byref(desc))
        workspace = torch.empty(ws_bytes // 4, dtype=torch.float32, device=x.device) if ws_bytes else None
    if any(ptr):
        _on(x.device, lib.ow_layer_norm_bwd, ctypes.byref(desc), dy.data_ptr(), dy_stride, *ptr,
            None if workspace is None else workspace.data_ptr(), ws_bytes)
    return grads


@torch.library.custom_op("omniwave_amd::layer_norm_fwd", mutates_args=())
def layer_norm_fwd(x: Tensor, weight: Tensor | None, bias: Tensor | None, eps: float) -> Tensor:
    """``layer_norm_hip``'s result."""
    return _run_layer_norm_forward(x, weight, bias, eps)


@layer_norm_fwd.register_fake
def _layer_norm_fwd_fake(x, weight, bias, eps):
    return x.new_empty(x.shape)


@torch.library.custom_op("omniwave_amd::layer_norm_bwd", mutates_args=())
def layer_norm_bwd(dy: Tensor, x: Tensor, weight: Tensor | None, bias: Tensor | None, eps: float,
                   want: list[bool]) -> tuple[Tensor, Tensor, Tensor]:
    """Gradients of x, weight and bias; empty where ``want`` is false."""
    grads = _run_layer_norm_backward(dy, x, weight, bias, eps, want)
    return tuple(x.new_empty(0) if g is None else g for g in grads)


@layer_norm_bwd.register_fake
def _layer_norm_bwd_fake(dy, x, weight, bias, eps, want):
    return tuple(x.new_empty(0) if t is None or not w else t.new_empty(t.shape) for t, w in zip((x, weight, bias), want))


def _layer_norm_setup_context(ctx, inputs, output):
    *tensors, eps = inputs
    ctx.save_for_backward(*tensors)
    ctx.eps = float(eps)


def _layer_norm_backward(ctx, dy):
    saved = ctx.saved_tensors  # once, as above
    want = [n and t is not None for n, t in zip(ctx.needs_input_grad, saved)]
    grads = layer_norm_bwd(dy, *saved, ctx.eps, want)
    return *[g if w else None for g, w in zip(grads, want)], None


layer_norm_fwd.register_autograd(_layer_norm_backward, setup_context=_layer_norm_setup_context)


def layer_norm_hip(x: Tensor, weight: Tensor | None = None, bias: Tensor | None = None, eps: float = 1e-6) -> Tensor:
    """``(x - mean) / sqrt(variance + eps) * weight + bias`` over the last dimension (``[..., C]``, C up to 8,192,
    float16, bfloat16 or float32, rows at any one distance), rounded once from fp32.  ``weight`` and ``bias`` ``[C]``, each
    may be left out and may have another dtype than ``x``.  Differentiable once in x, weight and bias."""
    glue = _native.glue()
    if glue is not None and _plain(x, weight, bias):
        y = glue.layer_norm(x, weight, bias, eps)
        if y is not None:
            return y
    # Everything else is checked, and goes through the operator.
    eps = float(eps)
    _layer_norm_ready(x, weight, bias, eps)
    return layer_norm_fwd(x, weight, bias, eps)
