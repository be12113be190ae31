"""Distillation on the GPU (``-m gpu``) against the formula in 64 bits.

Tolerances, in half steps U = 2^-24 of fp32.  A power exp2((x - m) log2(e) / T): the difference, the factor (the temperature
and the quotient are rounded) and their product move it by at most 4 U |x - m| / T, exp2, the reciprocal and two products
add 8 U; a sum of such positive terms (400 steps here at the outside: a thread's, six levels, four waves, parts) 400 U.  So p is
within (4 |x - m| / T + 420) U of itself and q likewise.  A gradient entry is within that times its p and the sum of its q,
plus 8 U of both.  A row's loss, T^2 (sum q ((t - mt) - (x - m)) / T - ln zt + ln z): 450 U and 4 U of its value for
each logarithm, and for each entry q's error and 900 U of the magnitudes of both differences.
"""

from __future__ import annotations

import sys

import pytest
import torch

from omniwave_amd import distillation_hip

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
U = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
GONE = -100


def announce(msg: str) -> None:
    print(f"\n[gpu-case] {msg}", file=sys.stderr, flush=True)


def formula(x, v, i, temp, ignore, reduction, up):
    """(loss, its allowance, gradient, its allowance) in 64 bits."""
    k, top = x.shape[-1], v.shape[-1]
    x, v, i = x.detach().double().reshape(-1, k), v.double().reshape(-1, top), i.reshape(-1, top)
    rows = len(x)
    given = (i != ignore) & (v != -float("inf"))
    counted = given.any(1)
    at = torch.where(given, i, 0)
    v = torch.where(given, v, -float("inf"))
    mt = torch.where(counted, v.amax(1) if top else 0.0, 0.0)[:, None]
    dt = torch.where(given, (v - mt) / temp, 0)
    q = torch.where(given, dt.exp(), 0)
    zt = q.sum(1, keepdim=True)
    zt = torch.where(counted[:, None], zt, 1)
    q = q / zt
    m = x.amax(1, keepdim=True)
    dx = (x - m) / temp
    p = dx.exp()
    z = p.sum(1, keepdim=True)
    p = p / z
    picked = torch.where(q > 0, dx.gather(1, at), 0)
    terms = q * (dt - picked)
    losses = temp ** 2 * (terms.sum(1) + z.log()[:, 0] - zt.log()[:, 0]) * counted
    slack = 900 + 4 * (z.log() + zt.log())[:, 0] + (q * (4 * dt.abs() + 900) * (dt.abs() + picked.abs())).sum(1)
    slack = (temp ** 2 * U * slack + 8 * U * losses.abs()) * counted
    n = counted.sum().item()
    up = up.double()
    if reduction == "none":
        loss, weight, up = losses, 1.0, up.reshape(-1, 1)
    else:
        weight = 1.0 / n if reduction == "mean" else 1.0
        loss = losses.sum() * weight
        slack = slack.sum() * weight + 4 * U * loss.abs()
    scale = up * weight * temp * counted[:, None]
    hit = torch.zeros(rows, k, dtype=torch.float64, device=x.device).scatter_add_(1, at, q)
    hit_err = torch.zeros_like(hit).scatter_add_(1, at, q * (4 * dt.abs() + 420))
    grad = scale * (p - hit)
    gslack = scale.abs() * U * (torch.where(p > 0, p * (4 * dx.abs() + 430), 0) + hit_err + 10 * hit)
    return loss, slack, grad, gslack


def check(x, v, i, temp=1.0, ignore=GONE, reduction="mean", up=None):
    x = x.detach().requires_grad_(True)
    loss = distillation_hip(x, v, i, temperature=temp, ignore_index=ignore, reduction=reduction)
    if up is None:
        up = torch.randn(x.shape[:-1] if reduction == "none" else (), device=DEV).abs() + 0.5
    (grad,) = torch.autograd.grad(loss, x, up)
    ref, slack, gref, gslack = formula(x, v, i, temp, ignore, reduction, up)
    assert loss.dtype == torch.float32 and loss.shape == (x.shape[:-1] if reduction == "none" else ())
    gap = (loss.detach().double().reshape(ref.shape) - ref).abs() - slack
    assert gap.max().item() <= 0, f"loss {gap.max().item()} past the bound"
    assert grad.dtype == x.dtype and grad.shape == x.shape
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 2.0 ** -149
    gap = (grad.double().reshape(gref.shape) - gref).abs() - gslack - torch.finfo(x.dtype).eps / 2 * gref.abs() * (1 + 2 ** -10) - tiny
    gap = gap - 2.0 ** -126 * up.abs().max().item() * max(1.0, temp)  # exp2 flushes results below fp32's normal range
    assert gap.max().item() <= 0, f"gradient {gap.max().item()} past the bound"
    return loss.detach(), grad


def make(rows, k, top, dtype, seed=0, scale=3.0, absent=0.0, empty=0.0, vtype=None):
    gen = torch.Generator().manual_seed(seed)
    teacher = torch.randn(rows, k, generator=gen) * scale
    x = (0.5 * teacher + torch.randn(rows, k, generator=gen) * scale).to(dtype)
    v, i = teacher.topk(top, 1)
    gone = (torch.rand(rows, top, generator=gen) < absent) | (torch.rand(rows, 1, generator=gen) < empty)
    gone[0] = False
    return x.to(DEV), v.to(vtype or dtype).to(DEV), torch.where(gone, GONE, i).to(DEV)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,k,top", [(1, 1, 1), (1, 2, 2), (3, 7, 3), (8, 1000, 8), (65, 1000, 100), (5, 4096, 64), (5, 4097, 65),
                                        (300, 5001, 33), (1, 50000, 500), (7, 21841, 1), (2, 200000, 128), (1100, 33, 33),
                                        (2100, 100, 7), (2100, 300, 20), (2100, 700, 1)])
def test_sizes(rows, k, top, dtype) -> None:
    announce(f"distillation rows={rows} k={k} top={top} {dtype}")
    x, v, i = make(rows, k, top, TYPES[dtype], seed=rows + k, absent=0.2, empty=0.1)
    check(x, v, i)
    check(x, v, i, temp=4.0)


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("temp", [0.5, 1.0, 3.0])
@pytest.mark.parametrize("vtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("k", [10, 9001])
def test_every_form(reduction, temp, vtype, k) -> None:
    announce(f"distillation reduction={reduction} T={temp} teacher {vtype} k={k}")
    x, v, i = make(9, k, 6, torch.float32, absent=0.3, vtype=TYPES[vtype])
    check(x, v, i, temp, reduction=reduction)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,k", [(6, 50), (6, 5000), (6, 40000), (2100, 50), (2100, 200)])
def test_a_class_with_several_entries(rows, k, dtype) -> None:
    announce(f"distillation repeated classes rows={rows} k={k} {dtype}")
    x, v, i = make(rows, k, 40, TYPES[dtype])
    i[0, 7] = i[0, 3]
    i[1] = i[1, 0]  # all of them
    i[2, 20:] = i[2, :20]
    i[3, ::2] = GONE
    i[3, 5] = i[3, 1]
    i[4, 39] = i[4, 0]
    i[5, 10:30] = k - 1
    i[-1, 1] = i[-1, 38]
    for reduction in ("mean", "none"):
        first = check(x, v, i, 2.0, reduction=reduction, up=torch.ones(rows if reduction == "none" else (), device=DEV))
        again = check(x, v, i, 2.0, reduction=reduction, up=torch.ones(rows if reduction == "none" else (), device=DEV))
        assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("rows,k,top", [(6, 50, 700), (5, 3000, 2999), (4, 40000, 8000), (2100, 200, 190)])
def test_long_lists_with_repeated_classes(rows, k, top) -> None:
    """One class twice, every class of the list eight times, and one class alone in the list."""
    announce(f"distillation long lists with repeated classes rows={rows} k={k} top={top}")
    x, v, _ = make(rows, max(k, top), top, torch.float32)
    x = x[:, :k].contiguous()
    gen = torch.Generator().manual_seed(1)
    i = torch.stack([torch.randperm(max(k, top), generator=gen)[:top] % k for _ in range(rows)])
    i[0, -1] = i[0, 0]
    i[1] = i[1, : (top + 7) // 8].repeat(8)[:top]
    i[2] = k // 2
    for reduction in ("mean", "none"):
        check(x, v, i.to(DEV), 1.5, reduction=reduction)


def test_a_student_that_is_its_teacher_and_all_classes() -> None:
    """Every class is an entry and both have the same logits: loss and gradient are rounding alone."""
    announce("distillation of itself")
    x, _, _ = make(7, 300, 1, torch.float32)
    i = torch.stack([torch.randperm(300) for _ in range(7)]).to(DEV)
    loss, grad = check(x, x.gather(1, i), i, 2.0)
    assert abs(loss.item()) <= 2e-4
    check(x + 1000.0, x.gather(1, i), i)


@pytest.mark.parametrize("k", [100, 9000, 40000])
def test_rows_left_out_and_entries_that_are_none(k) -> None:
    announce(f"distillation empty rows and -inf entries k={k}")
    x, v, i = make(8, k, 5, torch.float32)
    i[1] = GONE
    v[2] = -float("inf")
    v[3, 1:] = -float("inf")
    i[4, :4] = GONE
    v[5, 2], i[5, 3] = -float("inf"), GONE
    v[6] = torch.finfo(torch.float32).min  # lowest finite value: entries like any other
    x[1, 3] = float("nan")  # nobody looks at a row that is left out
    for reduction in ("mean", "sum"):
        y = x.detach().requires_grad_(True)
        loss = distillation_hip(y, v, i, reduction=reduction)
        (grad,) = torch.autograd.grad(loss, y)
        assert loss.isfinite() and grad.isfinite().all() and not grad[1].any()
    x[1, 3] = 0.0
    for reduction in ("none", "mean", "sum"):
        _, grad = check(x, v, i, 2.0, reduction=reduction)
        assert not grad[1:3].any() and grad[3].any()
    i[:] = GONE
    y = x.detach().requires_grad_(True)
    loss = distillation_hip(y, v, i)
    assert loss.isnan() and not torch.autograd.grad(loss, y)[0].any()
    assert distillation_hip(x, v, i, reduction="sum").item() == 0.0
    assert not distillation_hip(x, v, i, reduction="none").any()
    none = distillation_hip(x, v[:, :0], i[:, :0], reduction="none")
    assert none.shape == (8,) and not none.any()


def test_another_ignored_index() -> None:
    announce("distillation ignore_index")
    x, v, i = make(9, 30, 6, torch.float32)
    check(x, v, i, ignore=int(i[3, 2]))
    check(x, v, i, ignore=int(i[3, 2]), reduction="none")
    check(x, v, i, ignore=1 << 40)


@pytest.mark.parametrize("k", [60, 9000])
def test_rows_that_are_no_numbers(k) -> None:
    announce(f"distillation bad rows k={k}")
    x, v, i = make(12, k, 5, torch.float32)
    clean = check(x, v, i, reduction="none", up=torch.ones(12, device=DEV))
    i[1, 2], i[2, 0], i[3, 4] = k, -1, 1 << 62
    v[4, 1], v[5, 0] = float("nan"), float("inf")
    x[6, 7], x[7, k - 1] = float("nan"), float("inf")
    x[8] = -float("inf")
    y = x.detach().requires_grad_(True)
    losses = distillation_hip(y, v, i, reduction="none")
    (grad,) = torch.autograd.grad(losses.sum(), y)
    assert losses[1:9].isnan().all() and grad[1:9].isnan().all()
    for t, c in zip((losses.detach(), grad), clean):
        assert torch.equal(t[[0, 9, 10, 11]], c[[0, 9, 10, 11]])
    assert distillation_hip(x, v, i).isnan()
    i[1:9] = GONE
    assert distillation_hip(x, v, i).isfinite()


def test_masked_classes() -> None:
    announce("distillation masked classes")
    x, v, i = make(6, 90, 4, torch.float32)
    x[:, ::3] = -float("inf")
    i = i // 3 * 3 + 1
    i[:, 1] = (i[:, 0] + 1) % 90
    x[:, 1], x[:, 2] = 0.5, 0.25
    check(x, v, i)
    check(x, v, i, reduction="none")
    i[2, 0] = 0  # the teacher wants a class that the student rules out
    y = x.detach().requires_grad_(True)
    losses = distillation_hip(y, v, i, reduction="none")
    (grad,) = torch.autograd.grad(losses.sum(), y)
    assert losses[2].item() == float("inf") and losses[:2].isfinite().all() and grad.isfinite().all() and grad[2, 0] < 0


def test_large_logits_and_temperatures() -> None:
    announce("distillation large logits, temperatures")
    x, v, i = make(6, 500, 20, torch.float32, scale=30.0)
    x[1] *= 1e4
    x[2] += 1e5
    v[3] *= 1e3
    v[4] += 1e5
    check(x, v, i)
    check(x, v, i, 1000.0)
    check(x, v, i, 0.01, reduction="none")


def test_strides_and_leading_dimensions() -> None:
    announce("distillation strides")
    for dtype in (torch.bfloat16, torch.float32):
        x, v, i = make(24, 33, 5, dtype, absent=0.2)
        wide = torch.full((4, 6, 50), float("nan"), dtype=dtype, device=DEV)
        wide[..., 3:36] = x.reshape(4, 6, 33)
        v, i = v.reshape(4, 6, 5), i.reshape(4, 6, 5)
        got = check(wide[..., 3:36], v, i, 2.0, up=torch.ones((), device=DEV))
        want = check(x, v.reshape(24, 5), i.reshape(24, 5), 2.0, up=torch.ones((), device=DEV))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1].reshape(24, 33), want[1])
        check(wide[..., 3:36].transpose(0, 1), v.transpose(0, 1), i.transpose(0, 1), reduction="none")
        check(wide[0, 0, 3:36], v[0, 0], i[0, 0])
        check(x[:1].expand(24, 33), v.reshape(24, 5), i.reshape(24, 5))
        check(x, v.reshape(24, 5).flip(1), i.reshape(24, 5).flip(1), reduction="none", up=torch.ones((), device=DEV).expand(24))


def test_no_rows() -> None:
    announce("distillation of nothing")
    x = torch.zeros(0, 7, device=DEV, requires_grad=True)
    v, i = torch.zeros(0, 3, device=DEV), torch.zeros(0, 3, dtype=torch.int64, device=DEV)
    loss = distillation_hip(x, v, i)
    assert loss.isnan() and torch.autograd.grad(loss, x)[0].shape == (0, 7)
    assert distillation_hip(x, v, i, reduction="sum").item() == 0.0
    assert distillation_hip(x, v, i, reduction="none").shape == (0,)


def test_gradient_against_differences() -> None:
    """Central differences of the 64-bit loss: their own error is of order h^2 and 2^-52 / h."""
    announce("distillation differences")
    x, v, i = make(5, 40, 6, torch.float32)
    i[2, 3] = i[2, 1]
    one = torch.ones((), device=DEV)
    _, grad = check(x, v, i, 1.7, up=one)
    d = torch.randn(x.shape, dtype=torch.float64, generator=torch.Generator().manual_seed(1)).to(DEV)
    h = 1e-5
    value = lambda sign: formula(x.double() + sign * h * d, v, i, 1.7, GONE, "mean", one)[0].item()
    slope = (value(1) - value(-1)) / (2 * h)
    assert abs((grad.double() * d).sum().item() - slope) <= 1e-6 * (grad.double() * d).abs().sum().item() + 1e-9


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,k,top", [(16, 2048, 3), (16, 2049, 3), (17, 100, 9), (8, 4096, 70), (9, 4096, 70), (3, 16385, 70),
                                        (40, 16400, 17), (42, 16400, 17), (250, 8193, 5), (2047, 40, 5), (2048, 40, 5), (8193, 3, 3),
                                        (9000, 130, 4), (9001, 600, 65), (9000, 1100, 2), (140001, 7, 2), (8200, 4097, 3)])
def test_sizes_where_another_kernel_or_another_cut_begins(rows, k, top, dtype) -> None:
    announce(f"distillation rows={rows} k={k} top={top} {dtype}")
    x, v, i = make(rows, k, top, TYPES[dtype], seed=rows + k, absent=0.1, empty=0.1)
    for reduction in ("mean", "none"):
        check(x, v, i, 2.0, reduction=reduction)


@pytest.mark.parametrize("rows,k", [(8, 1000), (64, 1000), (3, 50001), (10000, 61)])
def test_same_bits_on_a_side_stream_in_a_graph_and_through_the_operator(rows, k) -> None:
    announce(f"distillation rerun, stream, graph, operator rows={rows} k={k}")
    from omniwave_amd.distillation import distillation_fwd

    x, v, i = make(rows, k, 10, torch.bfloat16, absent=0.1, empty=0.1)
    x.requires_grad_(True)

    def step():
        loss = distillation_hip(x, v, i, temperature=2.0)
        return loss.detach(), torch.autograd.grad(loss, x)[0]

    want = [t.clone() for t in step()]
    assert all(torch.equal(p, q) for p, q in zip(step(), want))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    loss, _ = distillation_fwd(x, v, i, 2.0, GONE, 2)
    assert torch.equal(loss, want[0]) and torch.equal(torch.autograd.grad(loss, x)[0], want[1])
    del loss
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for n in range(3):
        with torch.no_grad():
            x.mul_(0.9)
            i.copy_(i.roll(1, 0))
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, eager)), f"replay {n}"


def test_past_32_bit_offsets() -> None:
    announce("distillation of 2.3e9 logits")
    x, v, i = make(1000, 33001, 20, torch.bfloat16)
    small = x.clone().requires_grad_(True)
    losses = distillation_hip(small, v, i, reduction="sum")
    (want,) = torch.autograd.grad(losses, small)
    large = x.repeat(70, 1).requires_grad_(True)
    assert large.numel() > 1 << 31
    i = i.repeat(70, 1)
    i[:-1000] = GONE  # the last rows alone count
    loss = distillation_hip(large, v.repeat(70, 1), i, reduction="sum")
    (grad,) = torch.autograd.grad(loss, large)
    assert torch.equal(grad[-1000:], want) and not grad[:1000].any()
    assert abs(loss.item() - losses.item()) <= 1e-6 * losses.item()
