"""ctypes binding of libomniwave_amd.so (the C ABI declared in include/omniwave_amd.h)."""

from __future__ import annotations

import ctypes
import threading
from pathlib import Path

LIB_PATH = Path(__file__).resolve().parent / "libomniwave_amd.so"

OW_OK = 0
OW_ROUTE = {"local": 0, "shifted": 1, "radix": 2}
OW_DTYPE_F32, OW_DTYPE_BF16, OW_DTYPE_F16 = 0, 1, 2
OW_FUSE_NORM, OW_FUSE_RESIDUAL, OW_FUSE_FP8 = 1, 2, 4
OW_WEIGHTS_X3 = 8

_c_int32_p = ctypes.POINTER(ctypes.c_int32)


class OwPlan(ctypes.Structure):
    _fields_ = [
        ("height", ctypes.c_int32),
        ("width", ctypes.c_int32),
        ("channels", ctypes.c_int32),
        ("spatial_tile", ctypes.c_int32),
        ("channel_tile", ctypes.c_int32),
        ("route", ctypes.c_int32),
        ("radix_level", ctypes.c_int32),
        ("window", ctypes.c_int32),
        ("shift", ctypes.c_int32),
    ]


class OwBlockNorms(ctypes.Structure):
    _fields_ = [
        ("rows", ctypes.c_int64),
        ("rows_per_image", ctypes.c_int64),
        ("x_stride", ctypes.c_int64),
        ("delta_stride", ctypes.c_int64),
        ("x", ctypes.c_void_p),
        ("delta", ctypes.c_void_p),
        ("post_weight", ctypes.c_void_p),
        ("gate", ctypes.c_void_p),
        ("scale", ctypes.c_void_p),
        ("next_weight", ctypes.c_void_p),
        ("channels", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("post_dtype", ctypes.c_int32),
        ("gate_dtype", ctypes.c_int32),
        ("next_dtype", ctypes.c_int32),
        ("gate_per_image", ctypes.c_int32),
        ("eps", ctypes.c_float),
    ]


class OwLayerNorm(ctypes.Structure):
    _fields_ = [("rows", ctypes.c_int64), ("x_stride", ctypes.c_int64)]
    _fields_ += [(name, ctypes.c_void_p) for name in ("x", "weight", "bias")]
    _fields_ += [(name, ctypes.c_int32) for name in ("channels", "dtype", "weight_dtype", "bias_dtype")]
    _fields_ += [("eps", ctypes.c_float)]


class OwAdamwTensor(ctypes.Structure):
    _fields_ = [(name, ctypes.c_void_p) for name in ("param", "grad", "exp_avg", "exp_avg_sq", "exp_avg_scale",
                                                     "exp_avg_sq_scale", "master", "step")]
    _fields_ += [("numel", ctypes.c_int64), ("group", ctypes.c_int64)]


class OwAdamwGroup(ctypes.Structure):
    _fields_ = [(name, ctypes.c_double) for name in ("lr", "beta1", "beta2", "eps", "weight_decay")]
    _fields_ += [("lr_device", ctypes.c_void_p)]


class OwCrossEntropy(ctypes.Structure):
    _fields_ = [(name, ctypes.c_int64) for name in ("rows", "classes", "row_stride", "ignore_index")]
    _fields_ += [(name, ctypes.c_void_p) for name in ("logits", "target", "target_b", "mix")]
    _fields_ += [("mix_value", ctypes.c_float), ("smoothing", ctypes.c_float), ("dtype", ctypes.c_int32),
                 ("reduction", ctypes.c_int32)]


class OwDistillation(ctypes.Structure):
    _fields_ = [(name, ctypes.c_int64) for name in ("rows", "classes", "row_stride", "ignore_index")]
    _fields_ += [(name, ctypes.c_void_p) for name in ("logits", "teacher", "indices")]
    _fields_ += [(name, ctypes.c_int32) for name in ("top", "dtype", "teacher_dtype", "reduction")]
    _fields_ += [("temperature", ctypes.c_float)]


class OwGatedLinear(ctypes.Structure):
    _fields_ = [("rows", ctypes.c_int64), ("x_stride", ctypes.c_int64)]
    _fields_ += [(name, ctypes.c_void_p) for name in ("x", "gate_weight", "up_weight")]
    _fields_ += [(name, ctypes.c_int32) for name in ("channels", "hidden", "dtype")]


class OwGatedPlan(ctypes.Structure):
    _fields_ = [("whole", ctypes.c_int64), ("cut", ctypes.c_int64)]
    _fields_ += [(name, ctypes.c_int32) for name in ("tile_rows", "tile_cols", "parts")]


OW_GATED = {"forward": 0, "gates": 1, "dx": 2, "dw": 3}
OW_REDUCE = {"none": 0, "sum": 1, "mean": 2}
OW_ADAMW_CHUNK, OW_ADAMW_BLOCK = 4096, 256

_SIGNATURES = {
    "ow_version": (ctypes.c_int, []),
    "ow_last_error": (ctypes.c_char_p, []),
    "ow_plan_dims": (ctypes.c_int, [ctypes.POINTER(OwPlan), _c_int32_p, _c_int32_p]),
    "ow_route_build": (ctypes.c_int, [ctypes.POINTER(OwPlan), _c_int32_p, _c_int32_p]),
    "ow_packed_weight_bytes": (ctypes.c_size_t, [ctypes.c_int32] * 4),
    "ow_pack_weights": (
        ctypes.c_int,
        [ctypes.c_void_p] * 6 + [ctypes.c_int32, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int32]
        + [ctypes.c_int32] * 5 + [ctypes.c_void_p, ctypes.c_void_p],
    ),
    "ow_bwd_block_workspace": (ctypes.c_size_t, [ctypes.POINTER(OwPlan)] + [ctypes.c_int32] * 6),
    "ow_bwd_block": (
        ctypes.c_int,
        [ctypes.c_void_p] * 7 + [ctypes.c_int32] + [ctypes.c_void_p] * 4
        + [ctypes.POINTER(OwPlan), ctypes.c_int32, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32, ctypes.c_float]
        + [ctypes.c_void_p] * 3 + [ctypes.c_int32, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p],
    ),
    "ow_weights_x3_supported": (ctypes.c_int32, [ctypes.POINTER(OwPlan)]),
    "ow_packed_weight_bytes_x3": (ctypes.c_size_t, [ctypes.c_int32] * 3),
    "ow_pack_weights_x3": (
        ctypes.c_int,
        [ctypes.c_void_p] * 6 + [ctypes.c_int32, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int32]
        + [ctypes.c_int32] * 4 + [ctypes.c_void_p, ctypes.c_void_p],
    ),
    "ow_packed_weight_bytes_fp8": (ctypes.c_size_t, [ctypes.c_int32] * 3),
    "ow_pack_weights_fp8": (
        ctypes.c_int,
        [ctypes.c_void_p] * 6 + [ctypes.c_int32, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int32]
        + [ctypes.c_int32] * 5 + [ctypes.c_void_p, ctypes.c_void_p],
    ),
    "ow_rms_scale": (
        ctypes.c_int,
        [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_float, ctypes.c_int32,
         ctypes.c_void_p],
    ),
    "ow_fwd_workspace_bytes": (ctypes.c_size_t, [ctypes.POINTER(OwPlan), ctypes.c_int32, ctypes.c_int32]),
    "ow_bigemm_fwd": (
        ctypes.c_int,
        [
            ctypes.c_void_p, ctypes.c_void_p, ctypes.c_float,
            ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p, ctypes.c_void_p,
            ctypes.POINTER(OwPlan), ctypes.c_int32, ctypes.c_int32, ctypes.c_int32,
            ctypes.c_int32, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p,
        ],
    ),
    "ow_bigemm_fwd_rows": (
        ctypes.c_int,
        [
            ctypes.c_void_p, ctypes.c_void_p, ctypes.c_float,
            ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p,
            ctypes.POINTER(OwPlan), ctypes.c_int32, ctypes.c_int32, ctypes.c_int32,
            ctypes.c_int32, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p,
        ],
    ),
    "ow_bigemm_fwd_chain": (
        ctypes.c_int,
        [
            ctypes.c_void_p, ctypes.c_void_p, ctypes.c_float,
            ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p,
            ctypes.POINTER(OwPlan), ctypes.c_int32, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32,
            ctypes.c_void_p, ctypes.c_int32, ctypes.c_void_p, ctypes.POINTER(ctypes.c_int32),
            ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p,
        ],
    ),
    "ow_bigemm_fwd_scales": (
        ctypes.c_int,
        [
            ctypes.c_void_p, ctypes.c_void_p, ctypes.c_float,
            ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p, ctypes.c_void_p,
            ctypes.POINTER(OwPlan), ctypes.c_int32, ctypes.c_int32, ctypes.c_int32,
            ctypes.c_int32, ctypes.c_void_p, ctypes.c_void_p, ctypes.POINTER(ctypes.c_int32), ctypes.c_void_p,
            ctypes.c_size_t, ctypes.c_void_p,
        ],
    ),
    "ow_bigemm_fwd_drop": (
        ctypes.c_int,
        [
            ctypes.c_void_p, ctypes.c_void_p, ctypes.c_float,
            ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p, ctypes.c_void_p,
            ctypes.POINTER(OwPlan), ctypes.c_int32, ctypes.c_int32, ctypes.c_int32,
            ctypes.c_int32, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p,
        ],
    ),
    "ow_bigemm_fwd_noalloc": (
        ctypes.c_int,
        [
            ctypes.c_void_p, ctypes.c_void_p, ctypes.c_float,
            ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p, ctypes.c_void_p,
            ctypes.POINTER(OwPlan), ctypes.c_int32, ctypes.c_int32, ctypes.c_int32,
            ctypes.c_int32, ctypes.c_void_p,
        ],
    ),
    "ow_scale_samples": (
        ctypes.c_int,
        [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_int32,
         ctypes.c_void_p],
    ),
    "ow_route_s2d_rows": (ctypes.c_int, [ctypes.POINTER(OwPlan), ctypes.c_int32, _c_int32_p, _c_int32_p]),
    "ow_stem_fwd": (
        ctypes.c_int,
        [ctypes.c_void_p] * 3 + [ctypes.c_int32] * 5 + [ctypes.c_void_p],
    ),
    "ow_fold_weights": (
        ctypes.c_int,
        [ctypes.c_void_p] * 3 + [ctypes.c_int32, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p]
        + [ctypes.c_int32] * 5 + [ctypes.c_void_p] * 7,
    ),
    "ow_bwd_gather": (
        ctypes.c_int,
        [ctypes.c_void_p] * 5 + [ctypes.POINTER(OwPlan), ctypes.c_int32, ctypes.c_int32] + [ctypes.c_void_p] * 3,
    ),
    "ow_bwd_gate": (ctypes.c_int, [ctypes.c_void_p] * 6 + [ctypes.c_int64, ctypes.c_int32, ctypes.c_void_p]),
    "ow_bwd_scatter": (
        ctypes.c_int,
        [ctypes.c_void_p] * 3 + [ctypes.POINTER(OwPlan), ctypes.c_int32, ctypes.c_int32, ctypes.c_void_p,
                                 ctypes.c_void_p],
    ),
    "ow_bwd_rmsnorm": (
        ctypes.c_int,
        [ctypes.c_void_p] * 5 + [ctypes.c_int64, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32, ctypes.c_void_p],
    ),
    "ow_tile_mix": (
        ctypes.c_int, [ctypes.c_void_p] * 5 + [ctypes.c_int64, ctypes.c_int32, ctypes.c_int32, ctypes.c_void_p],
    ),
    "ow_tile_outer": (
        ctypes.c_int,
        [ctypes.c_void_p] * 3 + [ctypes.c_int32, ctypes.c_int64, ctypes.c_int32, ctypes.c_int32, ctypes.c_void_p],
    ),
    "ow_bwd_packed_bytes": (ctypes.c_size_t, [ctypes.c_int32] * 3),
    "ow_pack_bwd_weights": (
        ctypes.c_int,
        [ctypes.c_void_p] * 3 + [ctypes.c_int32, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p]
        + [ctypes.c_int32] * 5 + [ctypes.c_void_p, ctypes.c_void_p],
    ),
    "ow_bwd_fused_partials": (ctypes.c_int64, [ctypes.c_int64, ctypes.c_int32, ctypes.c_int32]),
    "ow_bwd_fused": (
        ctypes.c_int,
        [ctypes.c_void_p] * 6 + [ctypes.c_size_t] + [ctypes.c_void_p] * 5
        + [ctypes.c_int64, ctypes.c_int64, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32,
           ctypes.c_void_p],
    ),
    "ow_bwd_channel": (
        ctypes.c_int,
        [ctypes.c_void_p] * 6 + [ctypes.c_size_t] + [ctypes.c_void_p] * 6
        + [ctypes.c_int64, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32, ctypes.c_void_p],
    ),
    "ow_bwd_channel_partials": (ctypes.c_int64, [ctypes.c_int64, ctypes.c_int32]),
    "ow_bwd_channel2": (
        ctypes.c_int,
        [ctypes.c_void_p] * 8 + [ctypes.c_size_t] + [ctypes.c_void_p] * 2
        + [ctypes.c_int64, ctypes.c_int64, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32,
           ctypes.c_void_p],
    ),
    "ow_bwd_channel_routed": (
        ctypes.c_int,
        [ctypes.c_void_p] * 5 + [ctypes.c_int32] + [ctypes.c_void_p] * 4 + [ctypes.c_size_t] + [ctypes.c_void_p] * 6
        + [ctypes.c_int32, ctypes.c_int32, ctypes.c_void_p],
    ),
    "ow_bwd_channel2_routed": (
        ctypes.c_int,
        [ctypes.c_void_p] * 9 + [ctypes.c_size_t] + [ctypes.c_void_p] * 2 + [ctypes.c_int32]
        + [ctypes.c_void_p] * 2 + [ctypes.c_int64, ctypes.c_int32, ctypes.c_int32, ctypes.c_void_p],
    ),
    "ow_bwd_param_reduce64_partials": (ctypes.c_int64, [ctypes.c_int64, ctypes.c_int32, ctypes.c_int32]),
    "ow_bwd_param_reduce64": (
        ctypes.c_int,
        [ctypes.c_void_p] * 4 + [ctypes.c_size_t, ctypes.c_void_p, ctypes.c_int64, ctypes.c_int64, ctypes.c_int32,
                                 ctypes.c_int32, ctypes.c_int32, ctypes.c_void_p],
    ),
    "ow_bwd_param_reduce128_partials": (ctypes.c_int64, [ctypes.c_int64, ctypes.c_int32, ctypes.c_int32]),
    "ow_bwd_param_reduce128": (
        ctypes.c_int,
        [ctypes.c_void_p] * 7 + [ctypes.c_int64, ctypes.c_int64, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32,
                                 ctypes.c_void_p],
    ),
    "ow_small_to_f32": (ctypes.c_int, [ctypes.c_void_p] * 3 + [ctypes.c_int32, ctypes.c_void_p, ctypes.c_void_p]),
    "ow_bwd_x3_packed_bytes": (ctypes.c_size_t, [ctypes.c_int32] * 3),
    "ow_pack_bwd_x3": (
        ctypes.c_int,
        [ctypes.c_void_p] * 3 + [ctypes.c_int32] + [ctypes.c_void_p] * 3 + [ctypes.c_int32] * 4
        + [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p],
    ),
    "ow_bwd_x3_fits": (ctypes.c_int, [ctypes.c_int32] * 3),
    "ow_bwd_channel_x3_partials": (ctypes.c_int64, [ctypes.c_int64, ctypes.c_int32]),
    "ow_bwd_channel_x3": (
        ctypes.c_int,
        [ctypes.c_void_p] * 7 + [ctypes.c_size_t] + [ctypes.c_void_p] * 8 + [ctypes.c_int32] * 7
        + [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p, ctypes.c_void_p],
    ),
    "ow_bwd_param_reduce_x3_ranges": (ctypes.c_int64, [ctypes.c_int64, ctypes.c_int32]),
    "ow_bwd_param_reduce_x3": (
        ctypes.c_int,
        [ctypes.c_void_p] * 7 + [ctypes.c_int64, ctypes.c_int64] + [ctypes.c_int32] * 3 + [ctypes.c_void_p],
    ),
    "ow_sum_rows": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int64, ctypes.c_int64, ctypes.c_void_p, ctypes.c_void_p]),
    "ow_bwd_fused_routed": (
        ctypes.c_int,
        [ctypes.c_void_p] * 5 + [ctypes.c_int32] + [ctypes.c_void_p] * 4 + [ctypes.c_size_t] + [ctypes.c_void_p] * 5
        + [ctypes.c_int64, ctypes.c_int32, ctypes.c_int32, ctypes.c_void_p],
    ),
    "ow_block_norms_fwd": (ctypes.c_int, [ctypes.POINTER(OwBlockNorms)] + [ctypes.c_void_p] * 3),
    "ow_block_norms_bwd_workspace": (ctypes.c_size_t, [ctypes.POINTER(OwBlockNorms)]),
    "ow_block_norms_bwd": (
        ctypes.c_int,
        [ctypes.POINTER(OwBlockNorms), ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p, ctypes.c_int64]
        + [ctypes.c_void_p] * 6 + [ctypes.c_size_t, ctypes.c_void_p],
    ),
    "ow_layer_norm_fwd": (ctypes.c_int, [ctypes.POINTER(OwLayerNorm)] + [ctypes.c_void_p] * 2),
    "ow_layer_norm_bwd_workspace": (ctypes.c_size_t, [ctypes.POINTER(OwLayerNorm)]),
    "ow_layer_norm_bwd": (
        ctypes.c_int,
        [ctypes.POINTER(OwLayerNorm), ctypes.c_void_p, ctypes.c_int64] + [ctypes.c_void_p] * 4
        + [ctypes.c_size_t, ctypes.c_void_p],
    ),
    "ow_grad_norm_partials": (ctypes.c_int64, [ctypes.c_void_p, ctypes.c_int32]),
    "ow_grad_norm": (
        ctypes.c_int,
        [ctypes.c_void_p, ctypes.c_int32, ctypes.c_int32, ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p],
    ),
    "ow_adamw_step": (
        ctypes.c_int,
        [ctypes.c_void_p, ctypes.c_int32, ctypes.POINTER(OwAdamwGroup)] + [ctypes.c_int32] * 4
        + [ctypes.c_void_p, ctypes.c_int64, ctypes.c_double, ctypes.c_void_p, ctypes.c_void_p],
    ),
    "ow_cross_entropy_workspace": (ctypes.c_size_t, [ctypes.POINTER(OwCrossEntropy)]),
    "ow_cross_entropy_fwd": (
        ctypes.c_int, [ctypes.POINTER(OwCrossEntropy)] + [ctypes.c_void_p] * 5 + [ctypes.c_size_t, ctypes.c_void_p],
    ),
    "ow_cross_entropy_bwd": (ctypes.c_int, [ctypes.POINTER(OwCrossEntropy)] + [ctypes.c_void_p] * 5),
    "ow_distillation_workspace": (ctypes.c_size_t, [ctypes.POINTER(OwDistillation)]),
    "ow_distillation_fwd": (
        ctypes.c_int, [ctypes.POINTER(OwDistillation)] + [ctypes.c_void_p] * 5 + [ctypes.c_size_t, ctypes.c_void_p],
    ),
    "ow_distillation_bwd": (ctypes.c_int, [ctypes.POINTER(OwDistillation)] + [ctypes.c_void_p] * 5),
    "ow_gated_linear_kept": (ctypes.c_size_t, [ctypes.POINTER(OwGatedLinear)]),
    "ow_gated_linear_fwd_workspace": (ctypes.c_size_t, [ctypes.POINTER(OwGatedLinear)]),
    "ow_gated_linear_fwd": (
        ctypes.c_int, [ctypes.POINTER(OwGatedLinear)] + [ctypes.c_void_p] * 3 + [ctypes.c_size_t, ctypes.c_void_p],
    ),
    "ow_gated_linear_plan": (ctypes.c_int, [ctypes.POINTER(OwGatedLinear), ctypes.c_int32, ctypes.POINTER(OwGatedPlan)]),
    "ow_gated_linear_bwd_workspace": (ctypes.c_size_t, [ctypes.POINTER(OwGatedLinear)]),
    "ow_gated_linear_bwd": (
        ctypes.c_int,
        [ctypes.POINTER(OwGatedLinear), ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64] + [ctypes.c_void_p] * 4
        + [ctypes.c_size_t, ctypes.c_void_p],
    ),
    "ow_bwd_params": (
        ctypes.c_int,
        [ctypes.c_void_p] * 3 + [ctypes.c_int32, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p]
        + [ctypes.c_int32] * 4 + [ctypes.c_void_p] * 9,
    ),
}

_lock = threading.Lock()
_lib: ctypes.CDLL | None = None
_load_error: str | None = None


class NativeLibraryError(RuntimeError):
    """libomniwave_amd.so is missing or does not load."""


def _load() -> ctypes.CDLL | None:
    global _lib, _load_error
    if _lib is not None:  # set once, under the lock
        return _lib
    with _lock:
        if _lib is not None or _load_error is not None:
            return _lib
        if not LIB_PATH.exists():
            _load_error = f"{LIB_PATH.name} is not built (run omniwave_amd._build.build())"
            return None
        try:
            lib = ctypes.CDLL(str(LIB_PATH))
            for name, (restype, argtypes) in _SIGNATURES.items():
                fn = getattr(lib, name)
                fn.restype = restype
                fn.argtypes = argtypes
        except (OSError, AttributeError) as exc:
            _load_error = f"cannot load {LIB_PATH}: {exc}"
            return None
        _lib = lib
        return _lib


def load_error() -> str | None:
    """Why the library is unusable, or None when it loaded."""
    _load()
    return _load_error


def lib() -> ctypes.CDLL:
    handle = _load()
    if handle is None:
        raise NativeLibraryError(_load_error or "libomniwave_amd.so unavailable")
    return handle


_glue = None
_glue_error: str | None = None


def glue():
    """The module of the small operators' native calls, or None (``glue_error`` says why)."""
    global _glue, _glue_error
    if _glue is None and _glue_error is None:
        if _load() is None:
            _glue_error = _load_error
            return None
        try:
            from omniwave_amd import _glue as module
        except ImportError as exc:
            _glue_error = f"cannot load _glue.so (run omniwave_amd._build.build()): {exc}"
            return None
        _glue = module
    return _glue


def glue_error() -> str | None:
    glue()
    return _glue_error


def check(rc: int, what: str) -> None:
    """Raise the library's error text for a non-zero status."""
    if rc != OW_OK:
        msg = lib().ow_last_error().decode(errors="replace")
        exc = ValueError if rc == 1 else RuntimeError
        raise exc(f"{what} failed (status {rc}): {msg}")


def make_plan(height, width, channels, spatial_tile, channel_tile, route, radix_level, window=4, shift=2) -> OwPlan:
    return OwPlan(height, width, channels, spatial_tile, channel_tile, OW_ROUTE[route], radix_level, window, shift)


def exported_symbols() -> list[str]:
    return sorted(_SIGNATURES)
