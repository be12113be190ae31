"""Gated feed-forward product on the GPU (``-m gpu``) against the formula in 64 bits.

Tolerances, in half steps U = 2^-24 of fp32 and E of the type.  G and U are sums of K products: within (K + 64) U of
the sum of magnitudes (dG, dU below).  The sigmoid s of G is within (2 |G| + 8) U of itself, and moves by s (1 - s) dG.  So
h = G s U is off by at most |s U| dG + |G U| s (1 - s) dG + |G s| dU + (2 |G| + 16) U |h|, and half a step E of its type.
Backward, dU = dh G s is off by |dh| (s + |G| s (1 - s)) dG + (2 |G| + 16) U |dU|, dG = dh U f(G), f = s (1 + G (1 - s)), |f'| <= 1/2, by
|dh| (|f| dU + |U| dG / 2 + |U| (1 + |G|) (2 |G| + 10) U); both are rounded to the type (E). The other products take these errors
times the magnitudes of their other operands, and as many U as they have terms, 64 more.  A sigmoid below 2^-126, the
least normal fp32, is taken for 0 (its reciprocal and exp2 know no smaller ones): 2^-126 times its factors.  These are bounds for the worst
signs; as a whole, dx and the weights' gradients have two roundings that are independent of each other, each at most E:
their relative 2-norm error is below E sqrt(2 / 3), and E is asked.
"""

from __future__ import annotations

import sys

import pytest
import torch

from omniwave_amd import gated_linear_hip

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
U = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}


def announce(msg: str) -> None:
    print(f"\n[gpu-case] {msg}", file=sys.stderr, flush=True)


def close(got, ref, slack, what, whole=True):
    assert got.shape == ref.shape, what
    e = torch.finfo(got.dtype).eps / 2
    off = (got.detach().double() - ref).abs()
    worst = (off - e * ref.abs() - TINY[got.dtype] - slack).max().item() if off.numel() else -1.0
    assert worst <= 0, f"{what}: {worst} past the bound"
    if whole and got.dtype != torch.float32 and off.numel() >= 64:
        rel = (off.norm() / ref.norm()).item()
        assert rel <= e, f"{what}: {rel} as a whole"


def formula(x, wg, wu, dh):
    """{name: (result, allowance)} in 64 bits."""
    dtype = x.dtype
    e, tiny = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0, TINY[dtype]
    k = x.shape[-1]
    x, wg, wu = x.detach().double().reshape(-1, k), wg.detach().double(), wu.detach().double()
    g, u = x @ wg.T, x @ wu.T
    eg, eu = ((k + 64) * U * (x.abs() @ w.abs().T) for w in (wg, wu))
    s = torch.sigmoid(g)
    ds = s * (1 - s)
    h = g * s * u
    fast, least = (2 * g.abs() + 16) * U, 2.0 ** -126
    out = {"h": (h, (s * u).abs() * eg + (g * u).abs() * ds * eg + (g * s).abs() * eu + fast * h.abs() + least * (g * u).abs())}
    if dh is None:
        return out
    dh = dh.detach().double().reshape(h.shape)
    du, f = dh * g * s, s * (1 + g * (1 - s))
    dg = dh * u * f
    e_du = dh.abs() * (s + g.abs() * ds) * eg + fast * du.abs() + e * du.abs() + tiny + least * (dh * g).abs()
    e_dg = dh.abs() * (f.abs() * eu + u.abs() * eg / 2 + u.abs() * (1 + g.abs()) * (2 * g.abs() + 10) * U) + e * dg.abs() + tiny
    e_dg = e_dg + least * (dh * u).abs() * (1 + g.abs())
    n, m = wg.shape[0], len(x)
    a_dg, a_du, ax = dg.abs(), du.abs(), x.abs()
    out["dx"] = dg @ wg + du @ wu, (e_dg + (2 * n + 64) * U * a_dg) @ wg.abs() + (e_du + (2 * n + 64) * U * a_du) @ wu.abs()
    out["dgate"] = dg.T @ x, (e_dg + (m + 64) * U * a_dg).T @ ax
    out["dup"] = du.T @ x, (e_du + (m + 64) * U * a_du).T @ ax
    return out


def make(rows, c, hidden, dtype, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    normal = lambda scale, *shape: (torch.randn(shape, generator=gen, device=DEV) * scale).to(dtype)
    return normal(1.0, rows, c), normal(c ** -0.5, hidden, c), normal(c ** -0.5, hidden, c), normal(0.1, rows, hidden)


def check(x, wg, wu, dh, whole=True):
    ref = formula(x, wg, wu, dh)
    leaves = [t.detach().requires_grad_(True) for t in (x, wg, wu)]
    with torch.no_grad():
        plain = gated_linear_hip(x, wg, wu)
    h = gated_linear_hip(*leaves)
    assert h.dtype == x.dtype and h.shape == (*x.shape[:-1], wg.shape[0]) and torch.equal(h.detach(), plain)
    close(h.reshape(-1, wg.shape[0]), *ref["h"], "h", whole)
    grads = torch.autograd.grad(h, leaves, dh)
    for name, g, t in zip(("dx", "dgate", "dup"), grads, leaves):
        assert g.dtype == t.dtype and g.shape == t.shape
        close(g.reshape(-1, x.shape[-1]), *ref[name], name, whole)
    return [h.detach(), *grads]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 32, 33, 48, 64, 65, 127, 128, 129, 200])
@pytest.mark.parametrize("c,hidden", [(1, 1), (8, 16), (7, 5), (64, 33), (95, 190), (128, 256), (520, 72), (33, 8)])
def test_rows(rows, c, hidden, dtype) -> None:
    announce(f"gated rows={rows} c={c} hidden={hidden} {dtype}")
    check(*make(rows, c, hidden, TYPES[dtype], seed=rows + c))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows", [65, 127, 128, 129, 191, 192, 193, 255, 256, 257, 400])
@pytest.mark.parametrize("c,hidden", [(40, 4104), (95, 4101)])
def test_rows_of_tiles(rows, c, hidden, dtype) -> None:
    announce(f"gated tiles rows={rows} c={c} hidden={hidden} {dtype}")
    check(*make(rows, c, hidden, TYPES[dtype], seed=rows + c))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("c", [1, 2, 7, 8, 15, 16, 31, 32, 40, 63, 64, 65, 72, 96, 127, 128, 129, 136, 257])
@pytest.mark.parametrize("rows", [9, 6000])
def test_channels(rows, c, dtype) -> None:
    announce(f"gated rows={rows} c={c} {dtype}")
    check(*make(rows, c, 40, TYPES[dtype], seed=c))


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("hidden", [1, 3, 4, 8, 9, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300])
@pytest.mark.parametrize("rows", [5, 140, 6000])
def test_hidden(rows, hidden, dtype) -> None:
    announce(f"gated rows={rows} hidden={hidden} {dtype}")
    check(*make(rows, 48, hidden, TYPES[dtype], seed=hidden))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,c,hidden", [
    (16385, 40, 512),   # 256 x 256 tiles forward
    (16385, 37, 509),   # the same through registers
    (2049, 72, 1024),   # 128 x 128 tiles
    (2049, 71, 1023),
    (65537, 40, 16),    # 256 x 256 tiles in dx
    (65537, 41, 17),
    (100, 2816, 2896),  # 256 x 256 tiles in the weights' gradients
    (99, 2815, 2895),
    (9000, 128, 256),   # sums of many parts
    (33000, 256, 1100), # whole tiles and parts of others
    (300, 1408, 130),   # parts of both projections
    (300, 2064, 70),    # both products kept
    (300, 2049, 33),
    (1200, 1024, 200),  # 256 workgroups of the kernel for few tokens, and more
    (1300, 1024, 200),
    (129, 1030, 2100),
    (49, 264, 2050),    # few tokens: 32 a workgroup; then 16
    (50, 264, 1000),
    (4097, 1024, 64),
    (70, 4096, 130),
])
def test_every_tile(rows, c, hidden, dtype) -> None:
    announce(f"gated tiles rows={rows} c={c} hidden={hidden} {dtype}")
    check(*make(rows, c, hidden, TYPES[dtype]))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [6, 300, 2900])
def test_large_and_small_gates(rows, dtype) -> None:
    announce(f"gated large gates rows={rows} {dtype}")
    x, wg, wu, dh = make(rows, 64, 96, TYPES[dtype])
    check(x * 4, wg * 4, wu, dh)
    x[1] = 0
    wg[5] = 0
    check(x, wg, wu, dh)
    # far ends of the sigmoid: 0 and 1
    x[:, 0], wg[:, 0] = 100.0, torch.linspace(-3, 3, 96, device=DEV).to(x.dtype)
    h = gated_linear_hip(x, wg, wu)
    assert h.isfinite().all()
    check(x, wg, wu, dh, whole=False)


@pytest.mark.parametrize("rows", [10, 300, 3400])
@pytest.mark.parametrize("c", [64, 95])
def test_a_row_that_is_no_number_stays_in_its_row(rows, c) -> None:
    announce(f"gated NaN and inf rows={rows} c={c}")
    for dtype in (torch.bfloat16, torch.float32):
        x, wg, wu, dh = make(rows, c, 70, dtype)
        clean = check(x, wg, wu, dh)
        x[3, c - 1], x[7, 0] = float("nan"), float("inf")
        dh[5, 69] = float("nan")
        x.requires_grad_(True)
        h = gated_linear_hip(x, wg, wu)
        (dx,) = torch.autograd.grad(h, x, dh)
        rest = [i for i in range(rows) if i not in (3, 7)]
        assert torch.equal(h[rest], clean[0][rest]) and h[3].isnan().all() and not h[7].isfinite().any()
        rest.remove(5)
        assert torch.equal(dx[rest], clean[1][rest]) and dx[[3, 5]].isnan().all()
        # a weight's row stays with its value
        x = x.detach().clone()
        x[3], x[7] = 0.0, 0.0
        wu[4, 2] = float("nan")
        h = gated_linear_hip(x, wg, wu)
        assert h[:3, 4].isnan().all() and h[:, :4].isfinite().all() and h[:, 5:].isfinite().all()


@pytest.mark.parametrize("rows", [11, 150, 5601])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows_of_wider_tensors_at_odd_addresses(rows, dtype) -> None:
    announce(f"gated strides rows={rows} {dtype}")
    dtype = TYPES[dtype]
    x, wg, wu, dh = make(rows, 64, 48, dtype)
    want = check(x, wg, wu, dh)
    for begin in (1, 8):
        wide = torch.full((rows, 88), float("nan"), dtype=dtype, device=DEV)
        up = torch.full((rows, 72), float("nan"), dtype=dtype, device=DEV)
        wide[:, begin:begin + 64], up[:, begin:begin + 48] = x, dh
        got = check(wide[:, begin:begin + 64], wg, wu, up[:, begin:begin + 48])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    flat = torch.full((2 * 48 * 64 + 1,), float("nan"), dtype=dtype, device=DEV)
    flat[1:1 + 48 * 64], flat[1 + 48 * 64:] = wg.reshape(-1), wu.reshape(-1)  # as one buffer at an odd address holds them
    got = check(x, flat[1:1 + 48 * 64].view(48, 64), flat[1 + 48 * 64:].view(48, 64), dh)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    both = torch.cat([wg, wu])
    got = check(x, both[:48], both[48:], dh)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    check(x, wg.T.contiguous().T, both.reshape(2, 48, 64).permute(1, 0, 2)[:, 1], dh)
    # Sums of one random factor, times others: their errors are no average over independent ones.
    check(x[:1].expand(rows, 64), wg, wu, dh[:, :1].expand(rows, 48), whole=False)
    check(x, wg, wu, torch.full((), 0.25, dtype=dtype, device=DEV).expand(rows, 48), whole=False)
    check(x, wg, wg, dh)  # the same weight twice: gradients of each
    check(x[::2], wg, wu, dh[::2])
    cube = x[:rows // 2 * 2].reshape(2, rows // 2, 64)
    check(cube.transpose(0, 1), wg, wu, dh[:rows // 2 * 2].reshape(2, rows // 2, 48).transpose(0, 1))
    check(x[0], wg, wu, dh[0])


def test_the_same_weight_twice_adds_its_gradients() -> None:
    announce("gated shared weight")
    x, wg, _, dh = make(100, 64, 48, torch.float32)
    _, _, a, b = check(x, wg, wg, dh)
    wg.requires_grad_(True)
    (both,) = torch.autograd.grad(gated_linear_hip(x, wg, wg), wg, dh)
    assert torch.equal(both, a + b)


def test_nothing() -> None:
    announce("gated of nothing")
    for shape, hidden in (((0, 8), 4), ((2, 0, 8), 4), ((3, 8), 0), ((70, 0), 4), ((3, 0), 0)):
        x = torch.zeros(shape, device=DEV, requires_grad=True)
        wg, wu = (torch.ones(hidden, shape[-1], device=DEV, requires_grad=True) for _ in range(2))
        h = gated_linear_hip(x, wg, wu)
        assert h.shape == (*shape[:-1], hidden) and not h.any()
        grads = torch.autograd.grad(h, (x, wg, wu), torch.ones_like(h))
        assert all(g.shape == t.shape and not g.any() for g, t in zip(grads, (x, wg, wu)))


@pytest.mark.parametrize("rows", [7, 90, 8300])
def test_gradient_against_differences(rows) -> None:
    """Central differences of the formula in 64 bits: their own error is of order h^2 and 2^-52 / h."""
    announce(f"gated differences rows={rows}")
    x, wg, wu, dh = make(rows, 24, 20, torch.float32)
    got = check(x, wg, wu, dh)[1:]
    gen = torch.Generator().manual_seed(3)
    for n, grad in enumerate(got):
        v = torch.randn(grad.shape, generator=gen, dtype=torch.float64).to(DEV)

        def value(step):
            t = [q.double() + (step * v if k == n else 0) for k, q in enumerate((x, wg, wu))]
            return (torch.nn.functional.silu(t[0] @ t[1].T) * (t[0] @ t[2].T) * dh.double()).sum().item()

        slope = (value(1e-5) - value(-1e-5)) / 2e-5
        scale = (grad.double() * v).abs().sum().item()
        assert abs((grad.double() * v).sum().item() - slope) <= 2e-6 * scale + 1e-7


def test_leaves_that_need_no_gradient() -> None:
    announce("gated partial gradients")
    for rows, c in ((40, 64), (300, 95), (5600, 95)):
        x, wg, wu, dh = make(rows, c, 48, torch.bfloat16)
        full = check(x, wg, wu, dh)[1:]
        for n in range(3):
            t = [q.detach().clone() for q in (x, wg, wu)]
            t[n].requires_grad_(True)
            assert torch.equal(torch.autograd.grad(gated_linear_hip(*t), t[n], dh)[0], full[n])


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,c,hidden", [(200, 2056, 72), (257, 2049, 31), (1100, 2064, 640), (1, 1536, 1), (5, 1540, 300), (64, 1600, 40),
                                            (130, 1537, 90)])
def test_products_kept_and_formed_again(rows, c, hidden, dtype) -> None:
    """The backward's two ways to both products: the same sums, in other orders at most."""
    announce(f"gated kept products rows={rows} c={c} hidden={hidden} {dtype}")
    from omniwave_amd.gated import gated_linear_bwd, gated_linear_fwd

    x, wg, wu, dh = make(rows, c, hidden, TYPES[dtype])
    h, kept = gated_linear_fwd(x, wg, wu, True)
    plain, none = gated_linear_fwd(x, wg, wu, False)
    assert kept.numel() == 2 * rows * hidden and not none.numel() and torch.equal(h, plain)
    ref = formula(x, wg, wu, dh)
    for n, w in enumerate((wg, wu)):
        slack = (c + 64) * U * (x.double().abs() @ w.double().abs().T)
        assert ((kept.view(2, rows, hidden)[n].double() - x.double() @ w.double().T).abs() <= slack).all()
    for saved in (kept, none):
        for name, g in zip(("dx", "dgate", "dup"), gated_linear_bwd(dh, saved, x, wg, wu, [True] * 3)):
            close(g, *ref[name], name)


def test_sizes_that_are_not_known_while_compiling() -> None:
    announce("gated compiled with dynamic sizes")
    torch._dynamo.reset()
    fn = torch.compile(lambda *t: gated_linear_hip(*t), backend="aot_eager", dynamic=True)
    for rows in (80, 90, 30, 9000):
        x, wg, wu, dh = make(rows, 128, 24, torch.float32)
        leaves = [t.requires_grad_(True) for t in (x, wg, wu)]
        got = torch.autograd.grad(fn(*leaves), leaves, dh)
        assert all(torch.equal(a, b) for a, b in zip(got, torch.autograd.grad(gated_linear_hip(*leaves), leaves, dh)))


@pytest.mark.parametrize("rows,c,hidden", [(1, 256, 512), (49, 1024, 2048), (700, 128, 96), (3000, 200, 256)])
def test_same_bits_on_a_side_stream_in_a_graph_and_through_the_operator(rows, c, hidden) -> None:
    announce(f"gated rerun, stream, graph, operator rows={rows}")
    from omniwave_amd.gated import gated_linear_fwd

    x, wg, wu, dh = make(rows, c, hidden, torch.bfloat16)
    leaves = [t.requires_grad_(True) for t in (x, wg, wu)]

    def step(fn=gated_linear_hip):
        h = fn(x, wg, wu)
        return h.detach(), *torch.autograd.grad(h, leaves, dh)

    want = [t.clone() for t in step()]
    for fn in (gated_linear_hip, lambda *t: gated_linear_fwd(*t, True)[0]):
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
            x.mul_(0.9)
            wu.mul_(1.1)
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, eager)), f"replay {n}"


@pytest.mark.parametrize("rows,c,hidden", [(2200000, 1024, 8), (1100000, 16, 2048)])
def test_past_32_bit_offsets(rows, c, hidden) -> None:
    """x, or h and the gradients of both projections, past 2^31 values: copies of the same rows have the same results."""
    announce(f"gated past 2^31 values rows={rows} c={c} hidden={hidden}")
    period = 1000
    x, wg, wu, dh = make(period, c, hidden, torch.bfloat16)
    x.requires_grad_(True)
    h = gated_linear_hip(x, wg, wu)
    want = h.detach(), torch.autograd.grad(h, x, dh)[0]
    large = x.detach().repeat(rows // period, 1).requires_grad_(True)
    assert rows * max(c, hidden) > 1 << 31
    wg.requires_grad_(True)
    h = gated_linear_hip(large, wg, wu)
    dx, dwg = torch.autograd.grad(h, (large, wg), dh.repeat(rows // period, 1))
    assert dwg.isfinite().all()
    for got, ref in zip((h.detach(), dx), want):
        for n in (0, rows // period // 2, rows // period - 1):
            gap = (got[n * period:(n + 1) * period].double() - ref.double()).abs()
            assert (gap <= 2.0 ** -7 * ref.double().abs() + 1e-4).all()  # other tiles may add in another order
