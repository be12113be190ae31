"""Layer norm on the GPU (``-m gpu``) against the formula in 64 bits.

Tolerances, in half steps U = 2^-24 of fp32.  A sum over a row adds at most 8 values a thread and 10 levels: within
20 U of the sum of magnitudes.  The kernel's mean is off by at most F = 21 U mean|x|, so differences from it have magnitudes of at
most |d| + F, their rounding is U of that, and their mean, which is taken off again, is within 20 U of its terms: a difference
d = x - mu is within U A, A = 22 mean(|d| + F) + 3 (|d| + F); the root r of the variance within r U R, R = r^2 mean(|d| A) + 25 (first order; where the variance is
that small, eps bounds r).  A value y is then within U (|w| r (A + |d| R) + 6 (|w d r| + |b|)).  Backward, h = g w:
both means of the row carry 20 U of their magnitudes, d and r what they had.  A weight's gradient adds rows in chains of at
most 64 rows of a thread, 256 row slots and 2 x 32 partial rows and slices here: 400 U of the sum of magnitudes, and
what n = d r is off.  Every output is rounded once: half a step of its type, half the smallest subnormal of fp16.
"""

from __future__ import annotations

import sys

import pytest
import torch

from omniwave_amd import layer_norm_hip

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
U = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def announce(msg: str) -> None:
    print(f"\n[gpu-case] {msg}", file=sys.stderr, flush=True)


def close(got, ref, slack, what):
    assert got.shape == ref.shape, what
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0.0
    gap = (got.detach().double() - ref).abs() - torch.finfo(got.dtype).eps / 2 * ref.abs() - tiny - slack
    worst = gap.max().item() if gap.numel() else -1.0
    assert worst <= 0, f"{what}: {worst} past the bound"


def formula(x, w, b, eps, up):
    """(result, allowance) of y, and of dx, dweight and dbias, in 64 bits."""
    c = x.shape[-1]
    x, up = x.detach().double().reshape(-1, c), up.detach().double().reshape(-1, c)
    one = torch.ones((), dtype=torch.float64, device=x.device)
    w = one if w is None else w.detach().double()
    b = 0 * one if b is None else b.detach().double()
    mean = lambda t: t.mean(-1, keepdim=True)
    mu = mean(x)
    d = x - mu
    r = (mean(d * d) + eps).rsqrt()
    far = d.abs() + 21 * U * mean(x.abs())
    a = 22 * mean(far) + 3 * far
    rr = r * r * mean(d.abs() * a) + 25
    n = d * r
    out = {"y": (n * w + b, U * (w.abs() * r * (a + d.abs() * rr) + 6 * ((w * n).abs() + b.abs())))}
    h = up * w
    s1, s2 = mean(h), mean(h * d)
    s1_mag, s2_mag = mean(h.abs()), mean((h * d).abs())
    back = r * r * s2
    dx = r * (h - s1 - d * back)
    err = 2 * h.abs() + 21 * s1_mag + a * back.abs() + d.abs() * r * r * (20 * s2_mag + mean(h.abs() * a) + s2.abs() * (2 * rr + 6))
    out["dx"] = dx, U * (r * err + r * (h.abs() + s1_mag + (d * back).abs()) * (rr + 8))
    n_err = r * a + n.abs() * rr
    out["dweight"] = (up * n).sum(0), U * (up.abs() * (n_err + 400 * n.abs())).sum(0)
    out["dbias"] = up.sum(0), U * 400 * up.abs().sum(0)
    return out


def make(shape, dtype, wdtype, weight=True, bias=True, seed=0, mean=0.5):
    gen = torch.Generator().manual_seed(seed)
    c = shape[-1]
    x = (torch.randn(shape, generator=gen) + mean * torch.randn(c, generator=gen)).to(dtype).to(DEV)
    w = (torch.rand(c, generator=gen) + 0.5).to(wdtype).to(DEV)
    b = (torch.randn(c, generator=gen) * 0.1).to(wdtype).to(DEV)
    return x, w if weight else None, b if bias else None, torch.randn(shape, generator=gen).to(dtype).to(DEV)


def check(x, w, b, up, eps=1e-6):
    ref = formula(x, w, b, eps, up)
    leaves = {"dx": x, "dweight": w, "dbias": b}
    leaves = {k: t.detach().requires_grad_(True) for k, t in leaves.items() if t is not None}
    y = layer_norm_hip(leaves["dx"], leaves.get("dweight"), leaves.get("dbias"), eps=eps)
    assert y.dtype == x.dtype and y.shape == x.shape
    close(y.reshape(-1, x.shape[-1]), *ref["y"], "y")
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), up)))
    for name, g in grads.items():
        assert g.dtype == leaves[name].dtype and g.shape == leaves[name].shape
        close(g.reshape(-1, x.shape[-1]) if name == "dx" else g, *ref[name], name)
    return [y.detach(), *grads.values()]


@pytest.mark.parametrize("dtype,wdtype", [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f32", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("c", [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 33, 64, 95, 128, 200, 384, 512, 1000, 1024, 2047, 4100, 8191, 8192])
def test_channels_and_types(c, dtype, wdtype) -> None:
    announce(f"layer norm c={c} {dtype} weights {wdtype}")
    check(*make((2, 5, c), TYPES[dtype], TYPES[wdtype], seed=c))


@pytest.mark.parametrize("weight", [True, False])
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("c", [6, 96, 3000])
def test_every_form(weight, bias, dtype, c) -> None:
    announce(f"layer norm weight={weight} bias={bias} {dtype} c={c}")
    check(*make((3, 4, 7, c), TYPES[dtype], torch.float32, weight, bias))


@pytest.mark.parametrize("shape", [(128,), (1, 128), (1, 1, 7), (300, 64), (2000, 40), (7, 300, 128), (2223, 33), (30000, 3), (3000, 8),
                                   (1025, 1024), (70001, 16)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows(shape, dtype) -> None:
    announce(f"layer norm shape={shape} {dtype}")
    check(*make(shape, TYPES[dtype], torch.float32))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("c", [4, 24, 100, 1024])
def test_rows_that_fill_no_workgroup_without_eps(c, dtype) -> None:
    announce(f"layer norm eps=0 c={c} {dtype}")
    check(*make((3, 7, c), TYPES[dtype], torch.float32), eps=0.0)


@pytest.mark.parametrize("c", [95, 256, 2048])
def test_a_mean_far_above_the_deviations(c) -> None:
    announce(f"layer norm far mean c={c}")
    x, w, b, up = make((6, c), torch.float32, torch.float32, mean=0.0)
    check(x + 1000.0, w, b, up)
    check(x * 1e-3 + 10.0, w, b, up)


def test_constant_zero_large_and_small_rows() -> None:
    announce("layer norm constant, large, small rows")
    x, w, b, up = make((8, 100), torch.float32, torch.float32)
    x[0], x[1], x[2] = 0.0, 5.3, -1e4
    x[3] *= 1e15
    x[4] *= 1e-15
    check(x, w, b, up)


@pytest.mark.parametrize("c", [5, 8, 100, 2048])
def test_a_row_that_is_no_number_stays_in_its_row(c) -> None:
    announce(f"layer norm NaN and inf rows c={c}")
    for dtype in (torch.bfloat16, torch.float32):
        x, w, b, up = make((16, c), dtype, dtype)
        clean = check(x, w, b, up)
        x[3, c - 1], x[9, 0], x[12, c // 2] = float("nan"), float("inf"), float("-inf")
        x.requires_grad_(True)
        y = layer_norm_hip(x, w, b)
        (dx,) = torch.autograd.grad(y, x, up)
        rest = [i for i in range(16) if i not in (3, 9, 12)]
        assert torch.equal(y[rest], clean[0][rest]) and torch.equal(dx[rest], clean[1][rest])
        assert y[[3, 9, 12]].isnan().all() and dx[[3, 9, 12]].isnan().all()


def test_rows_of_wider_tensors_at_odd_addresses() -> None:
    announce("layer norm strided and unaligned rows")
    for dtype in (torch.bfloat16, torch.float32):
        for c in (3, 88):
            x, w, b, up = make((3, 11, c), dtype, torch.float32)
            wide = torch.full((2, 3, 11, c + 13), float("nan"), dtype=dtype, device=DEV)
            wide[0, ..., 1:c + 1], wide[1, ..., 4:c + 4] = x, up
            got = check(wide[0, ..., 1:c + 1], w, b, wide[1, ..., 4:c + 4])
            assert all(torch.equal(p, q) for p, q in zip(got, check(x, w, b, up)))
            check(x.transpose(0, 1), w, b, up.transpose(0, 1))
            check(x, w, b, up[:, :1].expand(3, 11, c))
            check(x, w, b, torch.full((), 0.5, dtype=dtype, device=DEV).expand(3, 11, c))
            check(x.expand(3, 11, c)[:, ::2], torch.ones(2 * c, device=DEV)[::2], b, up[:, ::2])


def test_nothing() -> None:
    announce("layer norm of nothing")
    for shape in ((0, 64), (2, 0, 64), (2, 4, 0)):
        x, w, b, up = (t.requires_grad_(True) for t in make(shape, torch.bfloat16, torch.float32))
        y = layer_norm_hip(x, w, b)
        assert y.shape == shape
        grads = torch.autograd.grad(y, (x, w, b), up)
        assert all(g.shape == t.shape and not g.any() for g, t in zip(grads, (x, w, b)))


def test_gradient_against_differences() -> None:
    """Central differences of the formula in 64 bits: their own error is of order h^2 and 2^-52 / h."""
    announce("layer norm differences")
    x, w, b, up = make((6, 40), torch.float32, torch.float32)
    got = dict(zip(("x", "w", "b"), check(x, w, b, up)[1:]))
    gen = torch.Generator().manual_seed(3)
    s = {"x": x, "w": w, "b": b}
    for name, grad in got.items():
        v = torch.randn(grad.shape, generator=gen, dtype=torch.float64).to(DEV)
        h = 1e-5

        def value(sign):
            t = {k: q.double() + (sign * h * v if k == name else 0) for k, q in s.items()}
            return (formula(t["x"], t["w"], t["b"], 1e-6, up)["y"][0] * up.double()).sum().item()

        slope = (value(1) - value(-1)) / (2 * h)
        have, scale = (grad.double() * v).sum().item(), (grad.double() * v).abs().sum().item()
        assert abs(have - slope) <= 1e-6 * scale + 1e-7, name


def test_leaves_that_need_no_gradient() -> None:
    announce("layer norm partial gradients")
    x, w, b, up = make((40, 128), torch.bfloat16, torch.float32)
    full = check(x, w, b, up)[1:]
    for n in range(3):
        t = [q.detach() for q in (x, w, b)]
        t[n].requires_grad_(True)
        assert torch.equal(torch.autograd.grad(layer_norm_hip(*t), t[n], up)[0], full[n])
        t[n].requires_grad_(False)
    t = [x.detach().requires_grad_(True), None, b]
    check(*t, up)


@pytest.mark.parametrize("shape", [(4, 333, 128), (49, 1024), (9, 8192)])
def test_same_bits_on_a_side_stream_in_a_graph_and_through_the_operator(shape) -> None:
    announce(f"layer norm rerun, stream, graph, operator {shape}")
    from omniwave_amd.norms import layer_norm_fwd

    x, w, b, up = make(shape, torch.bfloat16, torch.float32)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]

    def step(fn=layer_norm_hip):
        y = fn(x, w, b, 1e-6)
        return y.detach(), *torch.autograd.grad(y, leaves, up)

    want = [t.clone() for t in step()]
    for fn in (layer_norm_hip, layer_norm_fwd):
        assert all(torch.equal(p, q) for p, q in zip(step(fn), want))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for n in range(3):
        with torch.no_grad():
            x.add_(0.25)
            w.mul_(1.5)
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, eager)), f"replay {n}"


def test_past_32_bit_offsets() -> None:
    """2.25e9 values: 550 copies of the same rows give 550 copies of their results, to the bit."""
    announce("layer norm of 2.25e9 values")
    x, w, b, up = make((1, 4000, 1024), torch.bfloat16, torch.float32)
    x.requires_grad_(True)
    y = layer_norm_hip(x, w, b)
    want = y.detach(), torch.autograd.grad(y, x, up)[0]
    large = x.detach().expand(550, 4000, 1024).contiguous().requires_grad_(True)
    assert large.numel() > 1 << 31
    y = layer_norm_hip(large, w, b)
    got = y.detach(), torch.autograd.grad(y, large, up.expand(550, 4000, 1024))[0]
    for g, r in zip(got, want):
        for image in (0, 261, 262, 523, 524, 549):  # around 2^30 and 2^31 values, the last
            assert torch.equal(g[image], r[0])
