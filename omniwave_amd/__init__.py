"""omniwave_amd — MI355X-native (gfx950) backend for the OmniWeave BiGEMM operator.

Public API mirrors the reference package (omniweave/__init__.py:5-8): ``create_model``,
``create_model_from_config`` and ``bigemm``; plus the route plans and the HIP entry points.
"""

__version__ = "0.1.0"

from omniwave_amd.bigemm import bigemm, register_backend
from omniwave_amd.block import enable_fp8
from omniwave_amd.distillation import distillation_hip
from omniwave_amd.gated import gated_linear_hip
from omniwave_amd.hip import bigemm_block_hip, bigemm_delta_hip, hip_is_supported
from omniwave_amd.loss import cross_entropy_hip
from omniwave_amd.norms import block_norms_hip, layer_norm_hip, rms_norm_hip
from omniwave_amd.optim import AdamW
from omniwave_amd.registry import create_model, create_model_from_config
from omniwave_amd.routing import RoutePlan, build_route_plan, build_stage_schedule

__all__ = [
    "AdamW",
    "RoutePlan",
    "bigemm",
    "bigemm_block_hip",
    "bigemm_delta_hip",
    "block_norms_hip",
    "build_route_plan",
    "build_stage_schedule",
    "create_model",
    "create_model_from_config",
    "cross_entropy_hip",
    "distillation_hip",
    "enable_fp8",
    "gated_linear_hip",
    "hip_is_supported",
    "layer_norm_hip",
    "register_backend",
    "rms_norm_hip",
]
