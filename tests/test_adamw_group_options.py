"""Options of ``torch.optim.AdamW`` that change the update and that this optimizer has not are refused, wherever
they come in: in a group, in a saved state, written into a group between steps (on the CPU)."""

from __future__ import annotations

import copy

import pytest
import torch

from omniwave_amd import AdamW, optim

OTHER_UPDATES = [("maximize", True), ("amsgrad", True), ("differentiable", True), ("decoupled_weight_decay", False)]


def param():
    p = torch.nn.Parameter(torch.randn(6, 5))
    p.grad = torch.randn(6, 5)
    return p


@pytest.mark.parametrize("name,value", OTHER_UPDATES)
def test_other_updates_are_refused(name, value) -> None:
    p, q = param(), param()
    with pytest.raises(ValueError, match=name):
        AdamW([{"params": [p], name: value}])
    opt = AdamW([p])
    with pytest.raises(ValueError, match=name):
        opt.add_param_group({"params": [q], name: value})
    assert len(opt.param_groups) == 1
    opt.param_groups[0][name] = value
    with pytest.raises(ValueError, match=name):
        optim._hyper(opt.param_groups[0])  # what a step reads of its groups
    opt.param_groups[0][name] = not value
    optim._hyper(opt.param_groups[0])


@pytest.mark.parametrize("name,value", OTHER_UPDATES[:3])
def test_states_saved_under_another_update_are_refused(name, value) -> None:
    p = param()
    other = torch.optim.AdamW([p], lr=0.5, **{name: value})
    if name == "differentiable":
        saved = torch.optim.AdamW([p], lr=0.5)
        saved.step()
        saved = saved.state_dict()
        saved["param_groups"] = other.state_dict()["param_groups"]
    else:
        other.step()
        saved = other.state_dict()
    opt = AdamW([p])
    opt.state[p]["kept"] = 1
    groups = copy.deepcopy([{k: v for k, v in g.items() if k != "params"} for g in opt.param_groups])
    with pytest.raises(ValueError, match=name):
        opt.load_state_dict(saved)
    assert opt.state[p] == {"kept": 1}  # as it was
    assert [{k: v for k, v in g.items() if k != "params"} for g in opt.param_groups] == groups
    plain = copy.deepcopy(saved)
    for group in plain["param_groups"]:
        group[name] = not value
    opt.load_state_dict(plain)
    assert opt.param_groups[0]["lr"] == 0.5 and (opt.state[p]["step"] == 1).all()


def test_coupled_decay_of_a_saved_state_is_refused() -> None:
    p = param()
    other = torch.optim.AdamW([p])
    other.step()
    saved = other.state_dict()
    saved["param_groups"][0]["decoupled_weight_decay"] = False
    with pytest.raises(ValueError, match="decoupled_weight_decay"):
        AdamW([p]).load_state_dict(saved)


def test_options_that_change_nothing_are_taken() -> None:
    p = param()
    opt = AdamW([{"params": [p], "maximize": False, "amsgrad": False, "foreach": True, "capturable": True, "fused": None,
                  "differentiable": False, "decoupled_weight_decay": True}])
    p.grad = None
    opt.step()
