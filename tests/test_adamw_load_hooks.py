"""``AdamW.load_state_dict`` with hooks, and with a dictionary that it refuses (on the CPU)."""

from __future__ import annotations

import copy

import pytest
import torch

from omniwave_amd import AdamW


def optimizer(bits=32, seed=0):
    gen = torch.Generator().manual_seed(seed)
    params = [torch.nn.Parameter(torch.randn(shape, generator=gen)) for shape in ((70, 70), (33,))]
    opt = AdamW(params, state_bits=bits)
    for p in params:
        opt.state[p] = opt._adopt(p, dict(step=7, exp_avg=torch.randn(p.shape, generator=gen),
                                          exp_avg_sq=torch.rand(p.shape, generator=gen)))
    return opt, params


@pytest.mark.parametrize("bits", [32, 8])
def test_what_a_hook_before_the_load_returns_is_loaded(bits) -> None:
    source, _ = optimizer(bits)
    opt, params = optimizer(bits, seed=1)

    def other(_opt, state_dict):
        changed = copy.deepcopy(state_dict)
        for entry in changed["state"].values():
            entry["step"] = torch.full_like(entry["step"], 9)
            entry["exp_avg"] = torch.zeros(entry["exp_avg"].shape).to(entry["exp_avg"].dtype)
        changed["param_groups"][0]["lr"] = 0.25
        return changed

    handle = opt.register_load_state_dict_pre_hook(other)
    opt.load_state_dict(source.state_dict())
    assert opt.param_groups[0]["lr"] == 0.25
    for p in params:
        assert (opt.state[p]["step"] == 9).all() and not opt.state[p]["exp_avg"].float().any()
        opt._check_state(p)
    handle.remove()
    opt.load_state_dict(source.state_dict())
    assert all((opt.state[p]["step"] == 7).all() for p in params)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_hook_behind_the_load_has_the_last_word(bits) -> None:
    source, theirs = optimizer(bits)
    opt, params = optimizer(bits, seed=1)
    seen = []

    def after(opt):
        for p in params:
            opt._check_state(p)  # what it sees are the states as they are loaded
            seen.append({k: v.clone() for k, v in opt.state[p].items()})
            opt.state[p]["step"] = torch.full_like(opt.state[p]["step"], 11)

    opt.register_load_state_dict_post_hook(after)
    opt.load_state_dict(source.state_dict())
    for p, q, entry in zip(params, theirs, seen):
        assert entry.keys() == source.state[q].keys()
        for k, v in entry.items():
            assert v.dtype == source.state[q][k].dtype and torch.equal(v.float(), source.state[q][k].float())
        assert (opt.state[p]["step"] == 11).all()


def test_a_refused_dictionary_changes_nothing() -> None:
    source, _ = optimizer()
    opt, params = optimizer(seed=1)
    before = [{k: v.clone() for k, v in opt.state[p].items()} for p in params]
    bad = source.state_dict()
    bad["state"][1] = {"step": torch.tensor(3.0)}  # the second parameter's
    bad["param_groups"][0]["lr"] = 0.25
    for _ in range(2):
        with pytest.raises(ValueError, match="has no"):
            opt.load_state_dict(bad)
        assert opt.param_groups[0]["lr"] == 1e-3
        for p, entry in zip(params, before):
            assert all(torch.equal(opt.state[p][k], v) for k, v in entry.items())
    short = source.state_dict()
    short["param_groups"][0]["params"] = [0]
    with pytest.raises(ValueError, match="size"):
        opt.load_state_dict(short)
    opt.load_state_dict(source.state_dict())
    assert not torch.equal(opt.state[params[0]]["exp_avg"], before[0]["exp_avg"])


def test_loaded_states_are_copies() -> None:
    source, theirs = optimizer()
    opt, params = optimizer(seed=1)
    saved = source.state_dict()
    saved["state"][0]["exp_avg_sq"] = saved["state"][0]["exp_avg_sq"].bfloat16()
    opt.load_state_dict(saved)
    kept = theirs[0], source.state[theirs[0]]["exp_avg"].clone()
    for entry in opt.state.values():
        for t in entry.values():
            t.zero_()
    assert torch.equal(source.state[kept[0]]["exp_avg"], kept[1])
    assert (source.state[theirs[1]]["step"] == 7).all()


def test_the_load_makes_no_second_set_of_states(monkeypatch) -> None:
    source, _ = optimizer(bits=8)
    opt, params = optimizer(bits=8, seed=1)
    saved = source.state_dict()
    saved["state"]["of the run"] = {"best": 0.5}  # what belongs to no parameter stays what it is
    cast = []
    real = torch.Tensor.to
    monkeypatch.setattr(torch.Tensor, "to", lambda t, *a, **k: cast.append(k.get("dtype")) or real(t, *a, **k))
    opt.load_state_dict(saved)
    monkeypatch.undo()
    assert not [d for d in cast if d is not None]  # the base class would cast states to their parameter's dtype
    assert opt.state["of the run"] == {"best": 0.5}
    assert all(opt.state[p]["exp_avg"].dtype == torch.float8_e4m3fn for p in params[:1])
    assert len(saved["state"]) == 3 and saved["state"][0].keys() == source.state[next(iter(source.state))].keys()
