"""A block with ``post_norm`` whose tensors are made anew without their values (``to_empty``, as models made on the meta
device are) and then loaded is the block that was saved (on the CPU)."""

from __future__ import annotations

import copy

import pytest
import torch

import omniwave_amd
from omniwave_amd.block import OmniWeaveBlock


def poisoned(t, *args, **kwargs):
    out = torch.empty(t.shape, dtype=t.dtype, device="cpu")
    return out.fill_(float("nan")) if out.is_floating_point() else out


def block():
    return OmniWeaveBlock(height=8, width=8, dim=128, channel_tile=64, route="local", radix_level=0, post_norm=True)


@pytest.mark.parametrize("start", ["cpu", "meta"])
def test_the_ones_are_ones_again(start) -> None:
    saved = block()
    with torch.device(start):
        again = block()
    again._apply(poisoned)  # as to_empty, where what is there is not chance
    again.load_state_dict(saved.state_dict())
    assert torch.equal(again._ones, torch.ones(128)) and "_ones" not in saved.state_dict()
    assert again.plan.token_indices.device.type == "cpu"
    for other in (again.to(torch.bfloat16), copy.deepcopy(again)):
        assert torch.equal(other._ones.float(), torch.ones(128)) and other._ones.dtype == other.gamma.dtype


def test_a_model_made_without_values() -> None:
    kwargs = dict(post_norm=True, input_size=64)
    saved = omniwave_amd.create_model("omniweave_t", **kwargs)
    with torch.device("meta"):
        again = omniwave_amd.create_model("omniweave_t", **kwargs)
    again.to_empty(device="cpu")
    again.load_state_dict(saved.state_dict())
    for module in again.modules():
        if isinstance(module, OmniWeaveBlock):
            assert torch.equal(module._ones, torch.ones(module.dim))
