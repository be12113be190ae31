"""Norms around a block on the GPU (``-m gpu``) against a plain form in 64 bits.

Tolerances: every output is rounded once (half a step of its type, relative to the value; half the
smallest subnormal of fp16 below its range), after fp32 arithmetic.  A sum over a row has at most 8
values a thread (2 vectors of 4) and 10 levels, a value then about 10 operations of half a step 2^-24
each: 40 half steps of the magnitudes that enter it cover the forward, 120 the backward, which goes
through two sums after a rebuilt forward.  A weight's gradient adds rows in chains of at most 64 rows of a
thread, 32 row slots, 32 partial rows and 32 slices here: 320 half steps of the sum of magnitudes.
"""

from __future__ import annotations

import sys

import pytest
import torch

from omniwave_amd import block_norms_hip, rms_norm_hip

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
U = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def announce(msg: str) -> None:
    print(f"\n[gpu-case] {msg}", file=sys.stderr, flush=True)


def half_step(dtype, ref):
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    return torch.finfo(dtype).eps / 2 * ref.abs() + tiny


def close(got, ref, slack, what):
    assert got.dtype.is_floating_point and got.shape == ref.shape, what
    gap = (got.detach().double().cpu() - ref).abs()
    allowed = half_step(got.dtype, ref) + slack
    worst = (gap - allowed).max().item() if gap.numel() else -1.0
    assert worst <= 0, f"{what}: {worst} past the bound (largest gap {gap.max().item()})"


class Plain:
    """Forward and backward in 64 bits on the CPU, with the magnitudes that enter each value."""

    def __init__(self, x, delta, post, gate, scale, nextw, eps, dout, dnext):
        d = lambda t: None if t is None else t.detach().double().cpu()
        x, delta, post, gate, scale, nextw, dout, dnext = map(d, (x, delta, post, gate, scale, nextw, dout, dnext))
        b, c = x.shape[0], x.shape[-1]
        per = lambda t: t.reshape(b, *[1] * (x.dim() - 2), -1)
        one = torch.ones((), dtype=torch.float64)
        s = one if scale is None else per(scale)
        g = one if gate is None else (gate if gate.dim() == 1 else per(gate))
        w1 = one if post is None else post
        self.out, self.out_mag = x, x.abs()
        u = r1 = None
        if delta is not None:
            r1 = one if post is None else (delta.square().mean(-1, keepdim=True) + eps).rsqrt()
            u = delta * r1
            branch = s * g * w1 * u
            self.out, self.out_mag = x + branch, x.abs() + branch.abs()
        out = self.out
        if nextw is not None:
            r2 = (out.square().mean(-1, keepdim=True) + eps).rsqrt()
            self.next = out * r2 * nextw
            # an error of out moves r2 by at most its mean share
            spread = (self.out_mag * out.abs()).mean(-1, keepdim=True) * r2 * r2
            self.next_mag = nextw.abs() * r2 * (self.out_mag + out.abs() * spread) + self.next.abs()
        if dout is None and dnext is None:
            return
        grad = torch.zeros_like(x) if dout is None else dout
        mag = grad.abs()
        if dnext is not None:
            h = dnext * nextw
            back = (out * h).mean(-1, keepdim=True) * r2 * r2
            grad = grad + r2 * (h - out * back)
            back_mag = ((self.out_mag * h.abs()).mean(-1, keepdim=True) * r2 * r2) * (1 + spread)
            mag = mag + r2 * (h.abs() * (1 + spread) + self.out_mag * back_mag)
            self.dnw = self.over_rows(dnext * out * r2, nextw)
            self.dnw_mag = self.over_rows(dnext.abs() * r2 * self.out_mag * (1 + spread), nextw)
        self.dx, self.dx_mag = grad, mag
        if delta is None:
            return
        e, e_mag = grad * s, mag * s.abs()
        if gate is not None:
            self.dgate = self.over_rows(e * w1 * u, gate)
            self.dgate_mag = self.over_rows(e_mag * (w1 * u).abs(), gate)
        q, q_mag = e * g, e_mag * g.abs()
        if post is not None:
            self.dpost, self.dpost_mag = self.over_rows(q * u, post), self.over_rows(q_mag * u.abs(), post)
            h, h_mag = q * w1, q_mag * w1.abs()
            q = r1 * (h - u * (u * h).mean(-1, keepdim=True))
            q_mag = r1 * (h_mag + u.abs() * (u.abs() * h_mag).mean(-1, keepdim=True))
        self.ddelta, self.ddelta_mag = q, q_mag

    @staticmethod
    def over_rows(t, w):
        if w.dim() == 1:
            return t.reshape(-1, t.shape[-1]).sum(0)
        return t.reshape(t.shape[0], -1, t.shape[-1]).sum(1)


def make(shape, dtype, wdtype, post=True, gate="channel", scale=False, nxt=True, delta=True, seed=0):
    gen = torch.Generator().manual_seed(seed)
    b, c = shape[0], shape[-1]
    normal = lambda s, f=1.0: (torch.randn(s, generator=gen) * f).to(dtype).to(DEV)
    weight = lambda *s: (torch.rand(s, generator=gen) + 0.5).to(wdtype).to(DEV)
    t = {"x": normal(shape), "delta": normal(shape, 0.3) if delta else None,
         "post": weight(c) if post and delta else None,
         "gate": None if gate == "none" or not delta else weight(c) if gate == "channel" else weight(b, c),
         "scale": None, "next": weight(c) if nxt or not delta else None}
    if scale and delta:
        t["scale"] = ((torch.rand(b, generator=gen) > 0.3).float() / 0.7).to(DEV)
    t["dout"] = normal(shape) if delta else None
    t["dnext"] = normal(shape) if t["next"] is not None else None
    return t


LEAVES = ("x", "delta", "post", "gate", "next")


def call(t, eps=1e-6):
    if t["delta"] is None:
        return None, rms_norm_hip(t["x"], t["next"], eps=eps)
    return block_norms_hip(t["x"], t["delta"], post_weight=t["post"], gate=t["gate"], scale=t["scale"],
                           next_weight=t["next"], eps=eps)


def check(t, eps=1e-6, dout=True, dnext=True):
    """Forward and backward of ``t`` against the plain form."""
    ref = Plain(t["x"], t["delta"], t["post"], t["gate"], t["scale"], t["next"], eps, t["dout"] if dout else None,
                t["dnext"] if dnext else None)
    leaves = [n for n in LEAVES if t[n] is not None]
    for n in leaves:
        t[n] = t[n].detach().requires_grad_(True)
    out, nxt = call(t, eps)
    if out is not None:
        close(out, ref.out, 40 * U * ref.out_mag, "out")
    if nxt is not None:
        close(nxt, ref.next, 40 * U * ref.next_mag, "next")
    pairs = [(o, g) for o, g, on in ((out, t["dout"], dout), (nxt, t["dnext"], dnext)) if o is not None and g is not None and on]
    if not pairs:
        return out, nxt, {}
    grads = dict(zip(leaves, torch.autograd.grad([o for o, _ in pairs], [t[n] for n in leaves], [g for _, g in pairs],
                                                 allow_unused=True)))
    for name, attr, n in (("x", "dx", 120), ("delta", "ddelta", 120), ("post", "dpost", 320), ("gate", "dgate", 320),
                          ("next", "dnw", 320)):
        if name in grads:
            want = getattr(ref, attr, None)
            if want is None:  # the output that it enters has no gradient
                assert grads[name] is None or not grads[name].any()
                continue
            close(grads[name], want, n * U * getattr(ref, attr + "_mag"), attr)
    return out, nxt, grads


@pytest.mark.parametrize("dtype,wdtype", [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f32", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("c", [1, 3, 7, 8, 64, 95, 128, 200, 512, 1000, 1024, 2047, 4100, 8191, 8192])
def test_channels_and_types(c, dtype, wdtype) -> None:
    announce(f"norms c={c} {dtype} weights {wdtype}")
    check(make((2, 5, c), TYPES[dtype], TYPES[wdtype], scale=c % 2 == 0, seed=c))


@pytest.mark.parametrize("gate", ["none", "channel", "image"])
@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("nxt", [True, False])
@pytest.mark.parametrize("scale", [True, False])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_every_form(gate, post, nxt, scale, dtype) -> None:
    announce(f"norms gate={gate} post={post} next={nxt} scale={scale} {dtype}")
    check(make((3, 4, 7, 96), TYPES[dtype], torch.float32, post=post, gate=gate, scale=scale, nxt=nxt))


@pytest.mark.parametrize("shape", [(1, 1, 128), (1, 128), (5, 40), (300, 1, 64), (2000, 1, 40), (7, 300, 128), (2, 1111, 33),
                                   (1, 3000, 8)])
@pytest.mark.parametrize("gate", ["channel", "image"])
def test_rows_and_images(shape, gate) -> None:
    announce(f"norms shape={shape} gate={gate}")
    check(make(shape, torch.bfloat16, torch.float32, gate=gate, scale=True))


@pytest.mark.parametrize("c", [5, 64, 96, 1024])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_norm_alone(c, dtype) -> None:
    announce(f"norm alone c={c} {dtype}")
    check(make((4, 9, c), TYPES[dtype], TYPES[dtype], delta=False))


@pytest.mark.parametrize("dout,dnext", [(True, False), (False, True)])
def test_one_upstream_gradient(dout, dnext) -> None:
    announce(f"norms upstream dout={dout} dnext={dnext}")
    _, _, grads = check(make((2, 6, 128), torch.bfloat16, torch.bfloat16), dout=dout, dnext=dnext)
    if not dnext:
        assert grads["next"] is None or not grads["next"].any()


def test_zero_rows_of_the_delta_and_large_values() -> None:
    announce("norms zero rows, large values")
    t = make((2, 8, 128), torch.float32, torch.float32)
    t["delta"][0, :3] = 0
    t["x"][1, 2] = 0
    t["delta"][1, 2] = 0
    t["x"][0, 1] *= 1e15
    t["x"][1, 1] *= 1e-15
    check(t)


def test_a_row_that_is_no_number_stays_in_its_row() -> None:
    announce("norms NaN and inf rows")
    t = make((2, 8, 96), torch.bfloat16, torch.bfloat16)
    clean = [v.clone() for v in call(t)]
    t["x"][0, 3, 5] = float("nan")
    t["delta"][1, 4, 7] = float("inf")
    got = call(t)
    for g, r in zip(got, clean):
        rest = torch.ones(2, 8, dtype=torch.bool)
        rest[0, 3] = rest[1, 4] = False
        assert torch.equal(g[rest.to(DEV)], r[rest.to(DEV)])
        assert g[0, 3].isnan().any() and g[1, 4].isnan().any()


def test_rows_of_wider_tensors_at_odd_addresses() -> None:
    announce("norms strided and unaligned rows")
    for dtype in (torch.bfloat16, torch.float32):
        t = make((3, 11, 88), dtype, torch.float32)
        for i, name in enumerate(("x", "delta", "dout", "dnext")):
            wide = torch.full((3, 11, 101), float("nan"), dtype=dtype, device=DEV)
            wide[..., i + 1:i + 89] = t[name]
            t[name] = wide[..., i + 1:i + 89]
        check(t)


def test_upstream_gradients_of_a_sum() -> None:
    announce("norms expanded upstream gradients")
    t = make((2, 5, 64), torch.float32, torch.float32)
    t["dout"] = torch.full((), 0.5, device=DEV).expand(2, 5, 64)
    t["dnext"] = torch.ones(64, device=DEV).expand(2, 5, 64)
    check(t)
    t["dout"] = torch.randn(2, 64, 5, device=DEV).transpose(1, 2)
    t["dnext"] = torch.randn(5, 2, 64, device=DEV).transpose(0, 1)
    check(t)


def test_no_rows() -> None:
    announce("norms of nothing")
    for shape in ((0, 4, 64), (2, 0, 64), (2, 4, 0)):
        t = make(shape, torch.bfloat16, torch.float32, gate="image")
        for n in LEAVES:
            t[n].requires_grad_(True)
        out, nxt = call(t)
        assert out.shape == nxt.shape == shape
        grads = torch.autograd.grad((out, nxt), [t[n] for n in LEAVES], (t["dout"], t["dnext"]))
        assert all(g.shape == t[n].shape and not g.any() for g, n in zip(grads, LEAVES))


def test_gradient_against_differences() -> None:
    """Central differences of the 64-bit plain form along random directions: their own error, of order
    h^2 and 2^-52 / h, is far below the fp32 gradient's."""
    announce("norms differences")
    t = make((2, 6, 40), torch.float32, torch.float32, gate="image", scale=True)
    for n in LEAVES:
        t[n].requires_grad_(True)
    grads = torch.autograd.grad(call(t), [t[n] for n in LEAVES], (t["dout"], t["dnext"]))
    gen = torch.Generator().manual_seed(3)

    def value(name, v, h):
        s = {k: None if x is None else x.detach().double().cpu() for k, x in t.items()}
        s[name] = s[name] + h * v
        r = Plain(s["x"], s["delta"], s["post"], s["gate"], s["scale"], s["next"], 1e-6, None, None)
        return ((r.out * s["dout"]).sum() + (r.next * s["dnext"]).sum()).item()

    for name, grad in zip(LEAVES, grads):
        v = torch.randn(grad.shape, generator=gen, dtype=torch.float64)
        h = 1e-5
        slope = (value(name, v, h) - value(name, v, -h)) / (2 * h)
        got = (grad.double().cpu() * v).sum().item()
        scale = (grad.double().cpu().abs() * v.abs()).sum().item()
        assert abs(got - slope) <= 1e-6 * scale + 1e-7, f"{name}: {got} against {slope}"


def test_same_bits_again() -> None:
    announce("norms rerun")
    t = make((4, 333, 128), torch.bfloat16, torch.float32, scale=True)
    runs = []
    for _ in range(2):
        out, nxt, grads = check(dict(t))
        runs.append([out, nxt, *grads.values()])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_on_another_stream_and_in_a_graph() -> None:
    announce("norms side stream, captured forward and backward")
    t = make((4, 49, 512), torch.bfloat16, torch.float32, scale=True)
    for n in LEAVES:
        t[n].requires_grad_(True)

    def step():
        outs = call(t)
        return (*[o.detach() for o in outs], *torch.autograd.grad(outs, [t[n] for n in LEAVES], (t["dout"], t["dnext"])))

    want = [g.clone() for g in step()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(3):
        with torch.no_grad():
            t["x"].add_(0.25)
            t["post"].mul_(1.5)
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, eager)), f"replay {k}"


def test_leaves_that_need_no_gradient() -> None:
    announce("norms partial gradients")
    t = make((2, 6, 128), torch.bfloat16, torch.bfloat16)
    full = check(dict(t))[2]
    for only in LEAVES:
        s = {k: None if v is None else v.detach() for k, v in t.items()}
        s[only] = s[only].requires_grad_(True)
        (g,) = torch.autograd.grad(call(s), [s[only]], (s["dout"], s["dnext"]))
        assert torch.equal(g, full[only])


def test_the_operator_is_the_plain_call() -> None:
    announce("norms custom op")
    from omniwave_amd.norms import block_norms_fwd

    t = make((2, 6, 128), torch.bfloat16, torch.bfloat16, scale=True)
    plain = check(dict(t))
    for n in LEAVES:
        t[n] = t[n].detach().requires_grad_(True)
    out, nxt = block_norms_fwd(t["x"], t["delta"], t["post"], t["gate"], t["scale"], t["next"], 1e-6)
    assert torch.equal(out, plain[0]) and torch.equal(nxt, plain[1])
    grads = torch.autograd.grad((out, nxt), [t[n] for n in LEAVES], (t["dout"], t["dnext"]))
    assert all(torch.equal(g, plain[2][n]) for g, n in zip(grads, LEAVES))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(3, 7, 96), (2, 5, 1024), (5, 1, 33)])
def test_rows_that_fill_no_workgroup_without_eps(shape, dtype) -> None:
    """eps = 0: what a workgroup holds beside its last rows adds nothing to the weights' gradients."""
    announce(f"norms eps=0 {shape} {dtype}")
    check(make(shape, dtype, torch.float32, scale=True), eps=0.0)
    t = make(shape, dtype, torch.float32, scale=True, gate="image")
    check(dict(t), eps=0.0)
    for n in LEAVES:
        t[n] = t[n].detach().requires_grad_(True)
    t["scale"][0] = float("inf")  # an image's scale stays with it
    (g,) = torch.autograd.grad(call(t, eps=0.0), [t["gate"]], (t["dout"], t["dnext"]))
    assert g[1:].isfinite().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("c", [4096, 5000, 8192, 8190])
def test_wide_rows(c, dtype) -> None:
    announce(f"norms 2x400x{c} {dtype}")
    check(make((2, 400, c), dtype, torch.float32, scale=True))
