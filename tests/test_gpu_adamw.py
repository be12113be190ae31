"""AdamW on the GPU (``-m gpu``) against the formula in 64 bits.

Tolerances.  U = 2^-24 is half a step of fp32.  m and v are formed by three rounded operations from at
most two rounded constants, and with clipping from a gradient scaled by a rounded factor: 8 U of the
magnitudes that enter.  An update adds a root, two products, a sum and two divisions: 24 U of itself, and
the parameter's own decay 3 U of the parameter; a 16-bit parameter is rounded once more.  A value held
in 8 bits is off by half a step of e4m3fn, 2^-4 relative or 2^-10 scales below its normal range (a root above
zero that would be held as zero: 2^-9 scales), beside the same fp32 slack.
"""

from __future__ import annotations

import sys

import pytest
import torch

from omniwave_amd import AdamW, create_model
from omniwave_amd.optim import MIN_8BIT_VALUES, _decode

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
U = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SHAPES = [(1,), (3,), (), (255,), (256,), (257,), (16, 16), (4095,), (4096,), (4097,), (64, 129), (3, 64, 128), (70, 1001),
          (128, 1024)]


def announce(msg: str) -> None:
    print(f"\n[gpu-case] {msg}", file=sys.stderr, flush=True)


def make(shapes, dtype, seed=0, scale=1e-2):
    gen = torch.Generator().manual_seed(seed)
    params = [torch.nn.Parameter((torch.randn(s, generator=gen) * 0.1).to(dtype).to(DEV)) for s in shapes]
    return params, gen


def set_grads(params, gen, scale=1e-2):
    for i, p in enumerate(params):
        g = torch.randn(p.shape, generator=gen) * scale * 10.0 ** (i % 4 - 2)
        p.grad = g.to(p.dtype).to(DEV)


def snapshot(opt, params):
    """Parameters (masters where there are), first moments, second moments and steps in 64 bits."""
    out = []
    for p in params:
        e = opt.state.get(p) or {}
        zero = torch.zeros_like(p, dtype=torch.float64, device="cpu")
        if "exp_avg_sq_root" in e:
            m = _decode(e["exp_avg"], e["exp_avg_scale"]).double().cpu()
            v = _decode(e["exp_avg_sq_root"], e["exp_avg_sq_root_scale"]).double().cpu().square()
        else:
            m, v = (e[k].double().cpu() if e else zero.clone() for k in ("exp_avg", "exp_avg_sq"))
        w = e.get("master", p).detach().double().cpu()
        t = int(e["step"].reshape(-1)[0]) if e else 0
        out.append((w, m, v, t))
    return out


def held(value, exact, scale, fp32, what, least):
    """A value held in 8 bits beside the exact one."""
    s = scale.double().cpu().repeat_interleave(256)[:exact.numel()].reshape(exact.shape)
    step = torch.maximum(exact.abs() * 2.0 ** -4, s * 2.0 ** -10)
    if least:
        step = torch.where((exact > 0) & (exact < s * 2.0 ** -9), s * 2.0 ** -9, step)
        assert ((value > 0) == (exact > 0)).all(), what
    gap = (value - exact).abs() - step * (1 + 4 * U) - fp32
    assert gap.max().item() <= 0, f"{what}: {gap.max().item()} past the bound"


def check_step(opt, params, groups, max_norm=None, scales=None):
    """One step of ``opt`` against the formula from the states before it."""
    before = snapshot(opt, params)
    grads = [p.grad.double().cpu() for p in params]
    opt.step()
    torch.cuda.synchronize()
    coef = 1.0
    if max_norm is not None:
        norm = sum(g.square().sum() for g in grads).sqrt()
        assert abs(opt.grad_norm.double().cpu() - norm) <= 4 * U * norm
        coef = min(1.0, max_norm / (norm.item() + 1e-6))
    for i, (p, g, (w, m, v, t), (lr, wd)) in enumerate(zip(params, grads, before, groups)):
        what = f"parameter {i} {tuple(p.shape)} {p.dtype}"
        b1, b2, eps = 0.9, 0.999, 1e-8
        g, t = g * coef, t + 1
        m1 = b1 * m + (1 - b1) * g
        v1 = b2 * v + (1 - b2) * g * g
        m_mag = b1 * m.abs() + (1 - b1) * g.abs()
        root = v1.sqrt()
        denom = root / (1 - b2 ** t) ** 0.5 + eps
        update = lr / (1 - b1 ** t) * m1 / denom
        update_mag = lr / (1 - b1 ** t) * m_mag / denom
        w1 = w * (1 - lr * wd) - update
        slack = 24 * U * update_mag + 3 * U * w.abs() + 2.0 ** -149
        e = opt.state[p]
        assert (e["step"] == t).all(), what
        new = e.get("master", p).detach()
        gap = (new.double().cpu() - w1).abs() - slack - (torch.finfo(new.dtype).eps / 2 * (w1.abs() + slack) + (
            2.0 ** -25 if new.dtype == torch.float16 else 0.0))
        assert gap.max().item() <= 0, f"{what}: {gap.max().item()} past the bound"
        if "master" in e:
            assert torch.equal(p.detach(), e["master"].to(p.dtype)), what
        if "exp_avg_sq_root" in e:
            held(_decode(e["exp_avg"], e["exp_avg_scale"]).double().cpu(), m1, e["exp_avg_scale"], 8 * U * m_mag, what, False)
            held(_decode(e["exp_avg_sq_root"], e["exp_avg_sq_root_scale"]).double().cpu(), root, e["exp_avg_sq_root_scale"],
                 8 * U * root, what, True)
        else:
            tiny = 2.0 ** -149
            assert ((e["exp_avg"].double().cpu() - m1).abs() <= 8 * U * m_mag + tiny).all(), what
            assert ((e["exp_avg_sq"].double().cpu() - v1).abs() <= 8 * U * v1 + tiny).all(), what


@pytest.mark.parametrize("max_norm", [None, 0.05, 1e6])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype,master", [("f32", False), ("bf16", False), ("bf16", True), ("f16", True), ("f16", False)])
def test_steps(dtype, master, bits, max_norm) -> None:
    announce(f"adamw {dtype} master={master} bits={bits} max_norm={max_norm}")
    params, gen = make(SHAPES, TYPES[dtype])
    vectors = [p for p in params if p.dim() < 2]
    matrices = [p for p in params if p.dim() >= 2]
    opt = AdamW([{"params": matrices, "weight_decay": 0.1}, {"params": vectors, "lr": 3e-3}], lr=1e-3, weight_decay=0.0,
                state_bits=bits, master_weights=master, max_grad_norm=max_norm)
    groups = [(1e-3, 0.1) if p.dim() >= 2 else (3e-3, 0.0) for p in params]
    for _ in range(4):
        set_grads(params, gen)
        check_step(opt, params, groups, max_norm)
    for p in params:
        assert ("exp_avg_sq_root" in opt.state[p]) == (bits == 8 and p.numel() >= MIN_8BIT_VALUES)
        assert ("master" in opt.state[p]) == master


def test_more_tensors_than_a_launch_holds_and_more_groups() -> None:
    announce("adamw 400 tensors, 12 groups")
    shapes = [(1 + 37 * i % 900,) for i in range(400)]
    params, gen = make(shapes, torch.float32)
    opt = AdamW([{"params": params[i::12], "lr": 1e-3 * (i + 1)} for i in range(12)], weight_decay=0.01, max_grad_norm=1.0)
    groups = [(1e-3 * (i % 12 + 1), 0.01) for i in range(400)]
    for _ in range(2):
        set_grads(params, gen)
        check_step(opt, params, groups, 1.0)


def test_mixed_dtypes_make_one_norm() -> None:
    announce("adamw mixed dtypes")
    a, gen = make([(70, 70), (9,)], torch.float32)
    b, _ = make([(70, 71), (5, 5)], torch.bfloat16, seed=1)
    opt = AdamW(a + b, weight_decay=0.0, max_grad_norm=0.01, state_bits=8, master_weights=True)
    for _ in range(2):
        set_grads(a + b, gen)
        check_step(opt, a + b, [(1e-3, 0.0)] * 4, 0.01)


def test_values_beside_the_tensors_are_untouched() -> None:
    announce("adamw odd addresses")
    for dtype in (torch.float32, torch.bfloat16):
        for n in (1, 5, 255, 4097, 9000):
            flat = torch.full((n + 16,), 7.0, dtype=dtype, device=DEV)
            p = torch.nn.Parameter(flat[3:3 + n])
            gflat = torch.full((n + 16,), float("nan"), dtype=dtype, device=DEV)
            gflat[5:5 + n] = 0.01
            p.grad = gflat[5:5 + n]
            opt = AdamW([p], state_bits=8, master_weights=True, max_grad_norm=1.0)
            check_step(opt, [p], [(1e-3, 1e-2)], 1.0)
            assert (flat[:3] == 7).all() and (flat[3 + n:] == 7).all()
            # An update of 1e-3 is below half of bf16's step of 2^-5 at 7: there the masters move.
            assert not (opt.state[p].get("master", p.detach()) == 7).any()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_norm_that_is_not_finite_skips_the_step(bits, bad) -> None:
    announce(f"adamw skip {bad} bits={bits}")
    params, gen = make([(70, 70), (33,)], torch.float32)
    opt = AdamW(params, state_bits=bits, max_grad_norm=1.0)
    set_grads(params, gen)
    opt.step()
    kept = [p.detach().clone() for p in params]
    states = [{k: v.clone() for k, v in opt.state[p].items()} for p in params]
    set_grads(params, gen)
    params[1].grad[7] = bad
    opt.step()
    assert not torch.isfinite(opt.grad_norm)
    for p, q, s in zip(params, kept, states):
        assert torch.equal(p, q) and all(torch.equal(opt.state[p][k].float(), v.float()) for k, v in s.items())
    set_grads(params, gen)
    check_step(opt, params, [(1e-3, 1e-2)] * 2, 1.0)  # the second step that counts
    assert (opt.state[params[0]]["step"] == 2).all()


def test_large_gradients_have_a_finite_norm() -> None:
    announce("adamw large gradients")
    p = torch.nn.Parameter(torch.zeros(1000, device=DEV))
    p.grad = torch.full((1000,), 1e30, device=DEV)
    opt = AdamW([p], max_grad_norm=1.0)
    check_step(opt, [p], [(1e-3, 1e-2)], 1.0)


@pytest.mark.parametrize("bits", [32, 8])
def test_no_gradient_at_all_in_a_block(bits) -> None:
    announce(f"adamw zero gradients bits={bits}")
    p = torch.nn.Parameter(torch.randn(3000, 3, device=DEV))
    p.grad = torch.zeros_like(p)
    p.grad[100:105] = 1e-3
    opt = AdamW([p], state_bits=bits)
    for _ in range(3):
        check_step(opt, [p], [(1e-3, 1e-2)])
    assert torch.isfinite(p).all()


def test_tiny_second_moments_do_not_blow_up() -> None:
    """A root that is far below its block's largest is held at the least step and not as zero: the next
    update stays below lr times the ratio of the moments' growth."""
    announce("adamw 8-bit least root")
    p = torch.nn.Parameter(torch.zeros(4096, device=DEV))
    opt = AdamW([p], lr=1e-3, weight_decay=0.0, state_bits=8)
    g = torch.full((4096,), 1e-9, device=DEV)
    g[::256] = 1.0
    for _ in range(5):
        p.grad = g.clone()
        check_step(opt, [p], [(1e-3, 0.0)])
    assert p.abs().max() <= 5e-3 + 1e-6


def test_parameters_join_later_and_leave() -> None:
    announce("adamw changing sets")
    params, gen = make([(70, 70), (33,), (5, 5)], torch.float32)
    opt = AdamW(params)
    groups = [(1e-3, 1e-2)] * 3
    set_grads(params[:2], gen)
    check_step(opt, params[:2], groups)
    assert not opt.state.get(params[2])
    set_grads(params, gen)
    check_step(opt, params, groups)
    assert [int(opt.state[p]["step"][0]) for p in params] == [2, 2, 1]
    params[0].grad = None
    kept = params[0].detach().clone()
    check_step(opt, params[1:], groups)
    assert torch.equal(params[0], kept)
    opt.add_param_group({"params": [torch.nn.Parameter(torch.ones(7, device=DEV))], "lr": 0.1})
    extra = opt.param_groups[1]["params"][0]
    set_grads([*params, extra], gen)
    check_step(opt, [*params, extra], [*groups, (0.1, 1e-2)])


def test_moved_storage_and_replaced_states_are_followed() -> None:
    announce("adamw moved storage")
    params, gen = make([(70, 70), (33,)], torch.float32)
    opt = AdamW(params)
    set_grads(params, gen)
    opt.step()
    old = params[0].data
    params[0].data = old.clone()
    set_grads(params, gen)
    kept = old.clone()
    check_step(opt, params, [(1e-3, 1e-2)] * 2)
    assert torch.equal(old, kept)
    e = opt.state[params[1]]
    e["exp_avg"] = torch.ones_like(e["exp_avg"])
    set_grads(params, gen)
    check_step(opt, params, [(1e-3, 1e-2)] * 2)
    e["exp_avg_sq"] = torch.ones(3, device=DEV)
    with pytest.raises(ValueError, match="exp_avg_sq"):
        opt.step()


def test_strided_gradients_and_refused_ones() -> None:
    announce("adamw gradients' layouts")
    p = torch.nn.Parameter(torch.randn(40, 30, device=DEV))
    p.grad = torch.randn(30, 40, device=DEV).t()
    opt = AdamW([p], max_grad_norm=0.5)
    check_step(opt, [p], [(1e-3, 1e-2)], 0.5)
    p.grad = torch.ones((), device=DEV).expand(40, 30)
    check_step(opt, [p], [(1e-3, 1e-2)], 0.5)
    q = torch.nn.Parameter(torch.randn(4, 4, device=DEV))
    q.grad = torch.eye(4, device=DEV).to_sparse()
    with pytest.raises(RuntimeError, match="dense"):
        AdamW([q]).step()


def test_learning_rate_on_the_device() -> None:
    announce("adamw lr tensor")
    params, gen = make([(70, 70)], torch.float32)
    lr = torch.tensor(2e-3, device=DEV)
    opt = AdamW(params, lr=lr)
    set_grads(params, gen)
    check_step(opt, params, [(2e-3, 1e-2)])
    lr.fill_(5e-4)
    set_grads(params, gen)
    check_step(opt, params, [(5e-4, 1e-2)])
    opt.param_groups[0]["lr"] = torch.tensor(1e-3, device=DEV, dtype=torch.float64)
    with pytest.raises(ValueError, match="lr"):
        opt.step()


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps(bits) -> None:
    announce(f"adamw captured bits={bits}")
    shapes = [(70, 70), (33,), (3, 64, 128)]
    eager, gen = make(shapes, torch.bfloat16)
    held_, _ = make(shapes, torch.bfloat16)
    lr = torch.tensor(1e-3, device=DEV)
    kw = dict(lr=lr, state_bits=bits, master_weights=True, max_grad_norm=0.02)
    a, b = AdamW(eager, **kw), AdamW(held_, **kw)
    set_grads(held_, gen)
    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            b.step()

    def grads(k):
        g = torch.Generator().manual_seed(k)
        fresh = [(torch.randn(s, generator=g) * 0.01).to(torch.bfloat16).to(DEV) for s in shapes]
        if k == 3:
            fresh[1][0] = float("nan")
        for p, q, x in zip(eager, held_, fresh):
            p.grad = x.clone()
            q.grad.copy_(x)

    grads(0)
    a.step(), b.step()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        b.step()
    for k in range(1, 6):
        grads(k)
        lr.fill_(1e-3 / k)
        a.step()
        graph.replay()
        torch.cuda.synchronize()
        assert (a.grad_norm == b.grad_norm) or (k == 3 and a.grad_norm.isnan() and b.grad_norm.isnan())
        for p, q in zip(eager, held_):
            assert torch.equal(p, q)
            assert all(torch.equal(v.float(), b.state[q][n].float()) for n, v in a.state[p].items()), k
    assert (a.state[eager[0]]["step"] == 5).all()


def test_on_another_stream() -> None:
    announce("adamw side stream")
    params, gen = make([(128, 1024), (33,)], torch.float32)
    opt = AdamW(params, max_grad_norm=0.5)
    set_grads(params, gen)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        check_step(opt, params, [(1e-3, 1e-2)] * 2, 0.5)


def test_resumed_run_gives_the_same_bits() -> None:
    announce("adamw resume")
    runs = []
    for stop in (False, True):
        params, gen = make(SHAPES, torch.bfloat16)
        opt = AdamW(params, state_bits=8, master_weights=True, max_grad_norm=1.0)
        for k in range(6):
            if stop and k == 3:
                saved = opt.state_dict()
                opt = AdamW(params, state_bits=8, master_weights=True, max_grad_norm=1.0)
                opt.load_state_dict(saved)
            set_grads(params, gen)
            opt.step()
        runs.append([p.detach().clone() for p in params])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_a_model_follows_torch() -> None:
    """Three steps of OmniWeave-T beside torch.optim.AdamW: both round in fp32 alone, and every step's update
    is at most lr / sqrt(1 - b2) / (1 - b1) in size, so 3 steps differ by rounding only."""
    announce("adamw model")
    torch.manual_seed(0)
    ours = create_model("omniweave_t").to(DEV)
    theirs = create_model("omniweave_t").to(DEV)
    theirs.load_state_dict(ours.state_dict())
    a = AdamW(ours.parameters(), lr=1e-3, weight_decay=0.05)
    b = torch.optim.AdamW(theirs.parameters(), lr=1e-3, weight_decay=0.05, foreach=False)
    gen = torch.Generator(device=DEV).manual_seed(1)
    for _ in range(3):
        for p, q in zip(ours.parameters(), theirs.parameters()):
            p.grad = torch.randn(p.shape, generator=gen, device=DEV) * 1e-3
            q.grad = p.grad.clone()
        a.step(), b.step()
    for (name, p), q in zip(ours.named_parameters(), theirs.parameters()):
        # 3 steps of at most lr each way: 24 U of the updates and 3 U of the parameter per step and side
        bound = 6 * (24 * U * 1.1e-3 + 3 * U * p.detach().abs())
        assert ((p - q).detach().abs() <= bound).all(), name


def test_hooks_schedulers_closures_and_profiles_see_the_step() -> None:
    announce("adamw hooks, scheduler, closure, profiler")
    p = torch.nn.Parameter(torch.ones(300, device=DEV))
    opt = AdamW([p], lr=1e-2, weight_decay=0.0)
    schedule = torch.optim.lr_scheduler.StepLR(opt, 1, gamma=0.5)
    seen = []
    before = opt.register_step_pre_hook(lambda o, args, kwargs: seen.append("before"))
    after = opt.register_step_post_hook(lambda o, args, kwargs: seen.append("after"))
    p.grad = torch.ones_like(p)
    check_step(opt, [p], [(1e-2, 0.0)])
    assert seen == ["before", "after"]
    before.remove(), after.remove()
    schedule.step()
    check_step(opt, [p], [(5e-3, 0.0)])
    assert seen == ["before", "after"]

    def closure():
        opt.zero_grad()
        loss = (p * p).sum()
        loss.backward()
        return loss

    assert opt.step(closure).item() > 0 and (opt.state[p]["step"] == 3).all()
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as profile:
        opt.step()
    assert any("Optimizer.step#AdamW" in e.key for e in profile.key_averages())
    assert (opt.state[p]["step"] == 4).all()
