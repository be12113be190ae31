"""Cross-entropy on the GPU (``-m gpu``) against the formula in 64 bits.

Tolerances, in half steps U = 2^-24 of fp32.  A probability p = exp(x - m) / z: the difference and its
product with log2(e) are rounded, which moves the exponential by 2 U |x - m|; exp2, the reciprocal and two
products add 8 U; z adds its terms in at most 400 steps here (a thread's, six levels, four waves, parts), less than 64 U
for a pairwise-like sum of positive terms that each thread adds to a few hundred times, 400 U at the
outside.  So p is within (2 |x - m| + 420) U of itself, and a gradient entry within that times w p plus 4 U of
its other terms, and then half a step of its type.  A loss is within 440 U for ln z, 8 U of the magnitudes m -
x_a and the mean, whose sum adds at most 400 terms in a row: 420 U of the mean magnitude.
"""

from __future__ import annotations

import sys

import pytest
import torch

from omniwave_amd import cross_entropy_hip

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
U = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def announce(msg: str) -> None:
    print(f"\n[gpu-case] {msg}", file=sys.stderr, flush=True)


def formula(x, a, b, mix, s, ignore, reduction, up):
    """(loss, its allowance, gradient, its allowance) in 64 bits on the CPU."""
    k = x.shape[-1]
    x = x.detach().double().cpu().reshape(-1, k)
    a = a.cpu().reshape(-1)
    rows = x.shape[0]
    counted = a != ignore
    at = torch.where(counted, a, 0)
    w = torch.ones(rows, dtype=torch.float64)
    if b is not None:
        w = mix.double().cpu().reshape(-1) if isinstance(mix, torch.Tensor) else torch.full((rows,), float(mix), dtype=torch.float64)
    q = torch.full((rows, k), s / k, dtype=torch.float64)
    q.scatter_add_(1, at[:, None], (1 - s) * w[:, None])
    if b is not None:
        q.scatter_add_(1, b.cpu().reshape(-1, 1), (1 - s) * (1 - w)[:, None])
    m = x.amax(1, keepdim=True)
    p = (x - m).exp()
    z = p.sum(1, keepdim=True)
    p = p / z
    terms = torch.where(q > 0, q * (m - x), 0)
    losses = (terms.sum(1) + z.log()[:, 0]) * counted
    slack = (440 * U + 440 * U * terms.sum(1) + 440 * U * torch.where(q > 0, q * x.abs(), 0).sum(1) * (s > 0) + 2 * U * losses.abs()) * counted
    n = counted.sum().item()
    if reduction == "none":
        loss, weight, up = losses, 1.0, up.double().cpu().reshape(-1, 1)
    else:
        weight = 1.0 / n if reduction == "mean" else 1.0
        loss, slack, up = losses.sum() * weight, slack.sum() * weight, up.double().cpu()
        slack = slack + 4 * U * loss.abs()
    scale = up * weight * counted[:, None]
    grad = scale * (p - q)
    gslack = scale.abs() * (U * torch.where(p > 0, p * (2 * (m - x) + 420), 0) + 8 * U * q) + 8 * U * scale.abs() * p
    return loss, slack, grad, gslack


def check(x, a, b=None, mix=None, s=0.0, ignore=-100, reduction="mean", up=None):
    x = x.detach().requires_grad_(True)
    loss = cross_entropy_hip(x, a, target_b=b, mix=mix, label_smoothing=s, ignore_index=ignore, reduction=reduction)
    if up is None:
        up = torch.randn(a.shape if reduction == "none" else (), device=DEV).abs() + 0.5
    (grad,) = torch.autograd.grad(loss, x, up)
    ref, slack, gref, gslack = formula(x, a, b, mix, s, ignore, reduction, up)
    assert loss.dtype == torch.float32 and loss.shape == (a.shape if reduction == "none" else ())
    gap = (loss.detach().double().cpu().reshape(ref.shape) - ref).abs() - slack
    assert gap.max().item() <= 0, f"loss {gap.max().item()} past the bound"
    assert grad.dtype == x.dtype and grad.shape == x.shape
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 2.0 ** -149
    got = grad.double().cpu().reshape(gref.shape)
    gap = (got - gref).abs() - gslack - torch.finfo(x.dtype).eps / 2 * gref.abs() * (1 + 2 ** -10) - tiny
    # exp2 flushes results below fp32's normal range
    gap = gap - 2.0 ** -126 * up.abs().max().item()
    assert gap.max().item() <= 0, f"gradient {gap.max().item()} past the bound"
    return loss.detach(), grad


def make(rows, k, dtype, seed=0, scale=3.0, left_out=0.0):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, k, generator=gen) * scale).to(dtype).to(DEV)
    a = torch.randint(0, k, (rows,), generator=gen)
    b = torch.randint(0, k, (rows,), generator=gen)
    mix = torch.rand(rows, generator=gen)
    if left_out:
        out = torch.rand(rows, generator=gen) < left_out
        out[0] = False
        a[out] = -100
    return x, a.to(DEV), b.to(DEV), mix.to(DEV)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 2), (3, 7), (8, 1000), (65, 1000), (5, 4096), (5, 4097), (300, 5001), (1, 50000),
                                    (7, 21841), (2, 200000), (1100, 33)])
def test_sizes(rows, k, dtype) -> None:
    announce(f"xent rows={rows} k={k} {dtype}")
    x, a, b, mix = make(rows, k, TYPES[dtype], seed=rows + k, left_out=0.2)
    check(x, a)
    check(x, a, b, mix, s=0.1)


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("s", [0.0, 0.1, 1.0])
@pytest.mark.parametrize("two", ["one", "rows", "number", "first", "second"])
@pytest.mark.parametrize("k", [10, 9001])
def test_every_form(reduction, s, two, k) -> None:
    announce(f"xent reduction={reduction} smoothing={s} labels={two} k={k}")
    x, a, b, mix = make(9, k, torch.float32, left_out=0.3)
    mix = {"one": None, "rows": mix, "number": 0.3, "first": 1.0, "second": 0.0}[two]
    check(x, a, None if two == "one" else b, mix, s, reduction=reduction)


def test_the_same_label_twice_and_another_ignored_index() -> None:
    announce("xent equal labels, ignore_index")
    x, a, _, mix = make(9, 30, torch.float32)
    check(x, a, a.clone(), mix, 0.1)
    check(x, a, ignore=int(a[3]))
    check(x, a, ignore=int(a[3]), reduction="none")


def test_large_logits_and_a_sure_row() -> None:
    announce("xent large logits")
    x, a, _, _ = make(6, 500, torch.float32, scale=30.0)
    x[1] *= 1e4
    x[2] += 1e5
    x[3] = 0
    x[4] = 0
    x[4, a[4]] = 60.0
    check(x, a)
    check(x, a, reduction="none")


@pytest.mark.parametrize("k", [100, 9000])
def test_masked_classes_and_rows_that_are_no_numbers(k) -> None:
    announce(f"xent -inf, inf and NaN logits k={k}")
    x, a, b, _ = make(8, k, torch.float32)
    x[:, ::3] = float("-inf")
    a, b = a // 3 * 3 + 1, b // 3 * 3 + 2
    a, b = a.clamp(max=k - 2), b.clamp(max=k - 2)
    x.scatter_(1, a[:, None], 1.0), x.scatter_(1, b[:, None], 0.5)
    check(x, a, b, 0.3)
    check(x, a, a * 0, 1.0)  # the second label is masked and weighs nothing
    x[1] = float("-inf")
    x[2, 5] = float("inf")
    x[3, 7] = float("nan")
    a[4], a[5] = k, -1  # no such class
    x[6, :] = torch.finfo(torch.float32).min  # a mask of the lowest value over the whole row: uniform
    y = x.detach().requires_grad_(True)
    losses = cross_entropy_hip(y, a, reduction="none")
    (grad,) = torch.autograd.grad(losses.sum(), y)
    assert losses[1:6].isnan().all() and grad[1:6].isnan().any(1).all()
    assert torch.allclose(losses[6].double(), torch.tensor(float(k), device=DEV).double().log(), rtol=1e-5)
    assert torch.allclose(grad[6, a[6]], torch.tensor(1.0 / k - 1.0, device=DEV))
    clean = [0, 7]
    check(x[clean], a[clean], reduction="none")
    assert torch.equal(losses[clean], cross_entropy_hip(x[clean], a[clean], reduction="none"))
    a[1:6] = -100  # left-out rows do not spread what they hold
    y = x.detach().requires_grad_(True)
    loss = cross_entropy_hip(y, a)
    (grad,) = torch.autograd.grad(loss, y)
    assert loss.isfinite() and grad.isfinite().all() and not grad[1:6].any()


def test_no_rows_and_no_counted_rows() -> None:
    announce("xent of nothing")
    for shape in ((0, 10), (3, 0, 10)):
        x = torch.zeros(shape, device=DEV, requires_grad=True)
        a = torch.zeros(shape[:-1], dtype=torch.int64, device=DEV)
        for reduction in ("mean", "sum", "none"):
            loss = cross_entropy_hip(x, a, reduction=reduction)
            assert loss.shape == (a.shape if reduction == "none" else ())
            if reduction == "mean":
                assert loss.isnan()
            elif reduction == "sum":
                assert loss == 0
            assert torch.autograd.grad(loss.sum(), x)[0].shape == shape
    x = torch.randn(5, 10, device=DEV, requires_grad=True)
    a = torch.full((5,), -100, device=DEV)
    loss = cross_entropy_hip(x, a)
    assert loss.isnan() and not torch.autograd.grad(loss, x)[0].any()
    assert cross_entropy_hip(x, a, reduction="sum") == 0


def test_shapes_strides_and_addresses() -> None:
    announce("xent strided rows")
    gen = torch.Generator().manual_seed(0)
    a = torch.randint(0, 33, (4, 6), generator=gen).to(DEV)
    for dtype in (torch.float32, torch.bfloat16):
        wide = torch.randn(4, 6, 50, generator=gen).to(dtype).to(DEV)
        check(wide[..., 3:36], a)
        check(torch.randn(6, 4, 33, generator=gen).to(dtype).to(DEV).transpose(0, 1), a, reduction="none")
        check(torch.randn(33, generator=gen).to(dtype).to(DEV).expand(4, 6, 33), a)
        check(torch.randn(33, generator=gen).to(dtype).to(DEV), a[1, 2])
    losses = torch.randn(4, 6, device=DEV)
    check(wide[..., :33], a.t().contiguous().t(), a.flip(0), losses.sigmoid().t().contiguous().t(), 0.1)
    check(wide[..., :33], a, reduction="none", up=torch.ones((), device=DEV).expand(4, 6))


def test_gradient_against_differences() -> None:
    """Central differences of the 64-bit loss: their own error is of order h^2 and 2^-52 / h."""
    announce("xent differences")
    x, a, b, mix = make(5, 40, torch.float32)
    one = torch.ones((), device=DEV)
    _, grad = check(x, a, b, mix, 0.1, up=one)
    v = torch.randn(x.shape, dtype=torch.float64, generator=torch.Generator().manual_seed(1))
    h = 1e-5
    value = lambda sign: formula(x.double().cpu() + sign * h * v, a, b, mix, 0.1, -100, "mean", one)[0].item()
    slope = (value(1) - value(-1)) / (2 * h)
    got = (grad.double().cpu() * v).sum().item()
    assert abs(got - slope) <= 1e-6 * (grad.double().cpu().abs() * v.abs()).sum().item() + 1e-9


def test_the_loss_may_be_changed_in_place() -> None:
    announce("xent in-place")
    x, a, _, _ = make(8, 100, torch.float32)
    x.requires_grad_(True)
    loss = cross_entropy_hip(x, a)
    loss /= 4
    (grad,) = torch.autograd.grad(loss, x)
    (whole,) = torch.autograd.grad(cross_entropy_hip(x, a), x)
    assert torch.allclose(grad * 4, whole, rtol=1e-6, atol=0)


def test_same_bits_on_a_side_stream_in_a_graph_and_through_the_operator() -> None:
    announce("xent rerun, stream, graph, operator")
    from omniwave_amd.loss import cross_entropy_fwd

    for rows, k in ((64, 1000), (3, 50001)):
        x, a, b, mix = make(rows, k, torch.bfloat16, left_out=0.1)
        x.requires_grad_(True)

        def step():
            loss = cross_entropy_hip(x, a, target_b=b, mix=mix, label_smoothing=0.1)
            return loss.detach(), torch.autograd.grad(loss, x)[0]

        want = [t.clone() for t in step()]
        assert all(torch.equal(p, q) for p, q in zip(step(), want))
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            got = step()
        side.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        loss, _ = cross_entropy_fwd(x, a, b, mix, 1.0, 0.1, -100, 2)
        assert torch.equal(loss, want[0]) and torch.equal(torch.autograd.grad(loss, x)[0], want[1])
        del loss
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        for n in range(3):
            with torch.no_grad():
                x.mul_(0.9)
                a.copy_(a.roll(1))
            graph.replay()
            torch.cuda.synchronize()
            eager = step()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(held, eager)), f"replay {n}"


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,k", [(16, 2048), (16, 2049), (17, 100), (8, 4096), (9, 4096), (3, 16384), (3, 16385), (40, 16400),
                                    (42, 16400), (250, 8193), (1, 66000)])
def test_sizes_where_another_kernel_or_another_cut_begins(rows, k, dtype) -> None:
    """Sizes as above: a thread adds at most 16,400 / 256 terms where rows are not cut, 4,096 / 256 where they are."""
    announce(f"xent rows={rows} k={k} {dtype}")
    x, a, b, mix = make(rows, k, TYPES[dtype], seed=rows + k, left_out=0.2)
    for reduction in ("mean", "none"):
        check(x, a, b, mix, s=0.1, reduction=reduction)


def test_parts_of_a_row_without_a_number_above_minus_infinity() -> None:
    announce("xent masked parts")
    x, a, b, _ = make(6, 20000, torch.float32)
    x[0, :9000] = float("-inf")  # whole parts
    x[1, 9000:] = float("-inf")
    x[2, 4096:16384] = float("-inf")
    x[3] = float("-inf")
    x[4, 19999] = float("nan")
    x[5, 8000] = float("inf")
    a[:3] = torch.tensor([19999, 0, 19998], device=DEV)
    b[:3] = torch.tensor([9000, 8999, 4095], device=DEV)
    for reduction in ("none", "mean"):
        check(x[:3], a[:3], b[:3], 0.3, reduction=reduction)
    assert cross_entropy_hip(x, a, reduction="none")[3:].isnan().all()
    a[3:] = -100
    y = x.detach().requires_grad_(True)
    loss = cross_entropy_hip(y, a)
    (grad,) = torch.autograd.grad(loss, y)
    assert loss.isfinite() and grad.isfinite().all() and not grad[3:].any()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,k", [(2047, 40), (2048, 40), (8192, 3), (8193, 3), (8195, 9), (9000, 130), (9000, 260), (9001, 600),
                                    (9000, 1100), (140001, 7), (8200, 4097)])
def test_many_rows(rows, k, dtype) -> None:
    """Several rows a wave and a workgroup; a thread adds at most 4,097 / 64 terms."""
    announce(f"xent rows={rows} k={k} {dtype}")
    x, a, b, mix = make(rows, k, TYPES[dtype], seed=rows + k, left_out=0.2)
    first = check(x, a, b, mix, s=0.1)
    again = check(x, a, b, mix, s=0.1, up=torch.ones((), device=DEV))
    assert torch.equal(first[0], again[0])
    check(x, a, reduction="sum")
    check(x, a, b, mix, s=0.1, reduction="none")
    a[:] = -100
    y = x.detach().requires_grad_(True)
    loss = cross_entropy_hip(y, a)
    assert loss.isnan() and not torch.autograd.grad(loss, y)[0].any()


def test_many_rows_in_strides_with_bad_ones_and_in_a_graph() -> None:
    announce("xent many rows, strides, bad rows, graph")
    x, a, b, mix = make(10000, 61, torch.float32)
    wide = torch.zeros(10000, 70, device=DEV)
    wide[:, 5:66] = x
    wide.requires_grad_(True)

    def step():
        loss = cross_entropy_hip(wide[:, 5:66], a, target_b=b, mix=mix)
        return loss.detach(), torch.autograd.grad(loss, wide)[0]

    check(wide[:, 5:66], a, b, mix)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for n in range(3):
        with torch.no_grad():
            wide.mul_(0.9)
            a.copy_(a.roll(1))
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, eager)), f"replay {n}"
    x[77, 3], a[78] = float("nan"), 61
    losses = cross_entropy_hip(x, a, reduction="none")
    bad = losses.isnan()
    assert bad[77:79].all() and bad.sum() == 2 and cross_entropy_hip(x, a).isnan()
    a[77:79] = -100
    assert cross_entropy_hip(x, a).isfinite()
