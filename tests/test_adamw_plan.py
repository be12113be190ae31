"""AdamW's lists for the native calls are made anew where a parameter or a state lies as before but is no longer
what it was (another size, type, order): on the CPU, where the lists are made but nothing is launched."""

from __future__ import annotations

import pytest
import torch

from omniwave_amd import AdamW, _native, optim


@pytest.fixture(autouse=True)
def lists_on_the_cpu(monkeypatch):
    monkeypatch.setattr(optim, "gpu_reason", lambda t: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)


def param(*shape, dtype=torch.float32):
    p = torch.nn.Parameter(torch.randn(shape).to(dtype))
    p.grad = torch.randn(shape).to(dtype)
    return p


def plan_of(opt):
    glue = _native.glue()
    params = [p for group in opt.param_groups for p in group["params"]]
    lie = glue.gradients(params)
    assert lie is not None
    return optim._Plan(opt, glue, params, lie)


def current(plan, opt) -> bool:
    glue = _native.glue()
    params = [p for group in opt.param_groups for p in group["params"]]
    return plan.current(opt, glue, params, glue.gradients(params))


def change(p, data):
    """Another view at the address of ``p``, with a gradient that fits it."""
    assert data.data_ptr() == p.data_ptr()
    p.grad = None
    p.data = data
    p.grad = torch.ones(p.shape, dtype=p.dtype)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("how,text", [
    ("narrowed", "must be"), ("fewer rows", "must be"), ("wider", "must be"), ("transposed", "not contiguous"),
    ("reshaped", "must be"), ("retyped", "must be"), ("integers", "dtype"), ("negated", "negated view")])
def test_a_parameter_changed_in_place_is_refused(how, text, bits) -> None:
    store = torch.randn(2 * 64 * 64)
    p = torch.nn.Parameter(store[:64 * 64].view(64, 64))
    p.grad = torch.randn(64, 64)
    other = param(7)
    opt = AdamW([other, p], state_bits=bits)
    plan = plan_of(opt)
    assert current(plan, opt)
    d = p.data
    data = {"narrowed": lambda: d.view(-1)[:10], "fewer rows": lambda: d[:16], "wider": lambda: store.view(128, 64),
            "transposed": d.t, "reshaped": lambda: d.view(32, 128), "retyped": lambda: d.view(torch.bfloat16),
            "integers": lambda: d.view(torch.int32), "negated": lambda: torch._neg_view(d)}[how]()
    if how == "integers":
        with pytest.raises(RuntimeError):  # torch itself keeps a parameter floating point
            change(p, data)
        return
    change(p, data)
    if how == "negated":  # refused by every look
        with pytest.raises(ValueError, match=text):
            current(plan, opt)
    else:
        assert not current(plan, opt)
    with pytest.raises(ValueError, match=text):
        plan_of(opt)


def test_a_parameter_of_another_type_gets_its_own_kernel() -> None:
    p = param(40, dtype=torch.bfloat16)
    opt = AdamW([p])
    plan = plan_of(opt)
    change(p, p.data.view(torch.float16))
    assert not current(plan, opt)
    assert [kind.code for kind in plan_of(opt).kinds] == [_native.OW_DTYPE_F16]


@pytest.mark.parametrize("bits", [32, 8])
def test_a_state_changed_in_place_is_refused(bits) -> None:
    p = param(80, 80)
    opt = AdamW([p], state_bits=bits)
    plan = plan_of(opt)
    entry = opt.state[p]
    second = "exp_avg_sq" if bits == 32 else "exp_avg_sq_root"
    for name, data in (("exp_avg", entry["exp_avg"][:10]), (second, entry[second].t()), ("step", entry["step"][:1]),
                       ("exp_avg", entry["exp_avg"].view(torch.uint8)), ("step", entry["step"].view(torch.float32))):
        kept = entry[name]
        assert current(plan, opt)
        entry[name] = data
        assert data.data_ptr() == kept.data_ptr() and not current(plan, opt)
        with pytest.raises(ValueError, match=name):
            plan_of(opt)
        entry[name] = kept


def test_other_options_make_other_lists() -> None:
    p = param(80, 80, dtype=torch.bfloat16)
    opt = AdamW([p])
    plan = plan_of(opt)
    opt.master_weights = True
    assert not current(plan, opt)
    with pytest.raises(ValueError, match="master"):
        plan_of(opt)
    opt.master_weights, opt.state_bits = False, 8
    assert not current(plan, opt)
    with pytest.raises(ValueError, match="exp_avg"):
        plan_of(opt)
    opt.state_bits = 32
    assert current(plan, opt)


def test_shared_states_are_refused() -> None:
    p, q = param(80, 80), param(80, 80)
    opt = AdamW([p, q])
    plan_of(opt)
    kept = opt.state[q]
    opt.state[q] = opt.state[p]
    with pytest.raises(ValueError, match="states of parameters share"):
        plan_of(opt)
    opt.state[q] = {**kept, "exp_avg_sq": opt.state[p]["exp_avg_sq"]}
    with pytest.raises(ValueError, match="states of parameters share"):
        plan_of(opt)
    opt.state[q] = kept
    plan_of(opt)


def test_layouts() -> None:
    glue = _native.glue()
    t = torch.zeros(4, 4)
    views = [t, t[:2], t.t(), t.view(16), t.view(2, 8), t.view(torch.int32), t[None], t.double()]
    found = [glue.layouts([v]) for v in views]
    assert found[0] not in found[1:] and found[0] == glue.layouts([t])
    assert glue.layouts([t, t[:2]]) == found[0] + found[1] and glue.layouts([]) == b""
    views = [t, t[:2], t.t(), t.view(torch.int32), torch.zeros(4, 4)]
    states = [glue.state_layouts([{"a": v}]) for v in views]
    assert states[0] not in states[1:] and states[0] == glue.state_layouts([{"b": t}])
    assert glue.state_layouts([{"a": t}, {"b": t[:2]}, {}]) == states[0] + states[1]
    assert glue.state_layouts([{"a": 3}]) != glue.state_layouts([{"a": torch.zeros(())}])
    with pytest.raises(ValueError, match="negated"):
        glue.layouts([torch._neg_view(t)])
    with pytest.raises(ValueError, match="negated"):
        glue.state_layouts([{"a": torch._neg_view(t)}])
    for bad in (t, [1], None):
        with pytest.raises(TypeError):
            glue.layouts(bad)
        with pytest.raises(TypeError):
            glue.state_layouts(bad)
