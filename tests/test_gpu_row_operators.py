"""Layer norm, gated product and distillation as autograd sees them (``-m gpu``): hooks, recomputation, a second derivative,
compilation, calls at once, saved tensors that come back as others, and that the plain case is native."""

from __future__ import annotations

import sys
import threading

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from omniwave_amd import _native, distillation_hip, gated_linear_hip, layer_norm_hip

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def announce(msg: str) -> None:
    print(f"\n[gpu-case] {msg}", file=sys.stderr, flush=True)


def lnorm(dtype=torch.bfloat16, seed=0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(2, 30, 96, generator=gen).to(dtype).to(DEV)
    leaves = [x, torch.rand(96, generator=gen).to(DEV), torch.rand(96, generator=gen).to(DEV)]
    return [t.requires_grad_(True) for t in leaves], lambda *t: (layer_norm_hip(*t).float() * 0.5).sum()


def gated(dtype=torch.bfloat16, seed=0):
    gen = torch.Generator().manual_seed(seed)
    leaves = [torch.randn(*s, generator=gen).to(dtype).to(DEV) for s in ((2, 50, 96), (40, 96), (40, 96))]
    return [t.requires_grad_(True) for t in leaves], lambda *t: (gated_linear_hip(*t).float() * 0.5).sum()


def few(dtype=torch.float32, seed=0):
    leaves, fn = gated(dtype, seed)
    return [leaves[0].detach()[0, :9].requires_grad_(True), *leaves[1:]], fn


def kept(dtype=torch.float32, seed=0, rows=150):
    gen = torch.Generator().manual_seed(seed)
    leaves = [torch.randn(*s, generator=gen).to(dtype).to(DEV) for s in ((2, rows, 160), (40, 160), (40, 160))]
    return [t.requires_grad_(True) for t in leaves], lambda *t: (gated_linear_hip(*t).float() * 0.5).sum()


def tiles(dtype=torch.float32, seed=0):
    return kept(dtype, seed, 3000)


def distill(dtype=torch.bfloat16, seed=0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(33, 96, generator=gen).to(dtype).to(DEV).requires_grad_(True)
    v, i = torch.randn(33, 96, generator=gen).topk(7, 1)
    v, i = v.to(DEV), i.to(DEV)
    return [x], lambda x: distillation_hip(x, v, i, temperature=2.0)


CASES = {"lnorm": lnorm, "gated": gated, "few": few, "kept": kept, "tiles": tiles, "distill": distill}


@pytest.fixture(params=sorted(CASES))
def case(request):
    announce(f"row operator {request.param}")
    return CASES[request.param]()


def test_plain_calls_are_native(case, monkeypatch) -> None:
    leaves, fn = case
    glue, calls = _native.glue(), []

    class Counted:
        def __getattr__(self, name):
            def call(*args):
                result = getattr(glue, name)(*args)
                calls.append(result is not None)
                return result
            return call

    monkeypatch.setattr(_native, "glue", lambda: Counted())
    fn(*leaves).backward()
    with torch.inference_mode():
        fn(*leaves)
    assert len(calls) == 2 and all(calls)


def test_without_the_native_module(case, monkeypatch) -> None:
    leaves, fn = case
    want = [fn(*leaves), *torch.autograd.grad(fn(*leaves), leaves)]
    monkeypatch.setattr(_native, "glue", lambda: None)
    for a, b in zip(want, [fn(*leaves), *torch.autograd.grad(fn(*leaves), leaves)]):
        assert torch.equal(a, b)


def test_twice_through_a_kept_graph(case) -> None:
    leaves, fn = case
    loss = fn(*leaves)
    first = torch.autograd.grad(loss, leaves, retain_graph=True)
    for a, b in zip(first, torch.autograd.grad(loss, leaves)):
        assert torch.equal(a, b)


def test_saved_on_the_cpu_and_recomputed(case) -> None:
    leaves, fn = case
    want = torch.autograd.grad(fn(*leaves), leaves)
    with torch.autograd.graph.save_on_cpu():
        loss = fn(*leaves)
    for a, b in zip(torch.autograd.grad(loss, leaves), want):
        assert torch.equal(a, b)
    for t in leaves:
        t.grad = None
    checkpoint(fn, *leaves, use_reentrant=False).backward()
    for t, b in zip(leaves, want):
        assert torch.equal(t.grad, b)


def test_a_changed_input_is_noticed(case) -> None:
    leaves, fn = case
    loss = fn(*leaves)
    with torch.no_grad():
        leaves[0].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(loss, leaves)


def test_a_second_derivative_is_refused(case) -> None:
    leaves, fn = case
    grads = torch.autograd.grad(fn(*leaves), leaves, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        sum(g.float().square().sum() for g in grads).backward()


def test_no_graph_without_need(case) -> None:
    leaves, fn = case
    assert fn(*leaves).grad_fn is not None
    assert fn(*[t.detach() for t in leaves]).grad_fn is None
    with torch.no_grad():
        assert not fn(*leaves).requires_grad
    with torch.inference_mode():
        assert fn(*leaves).is_inference()


def test_compiled(case) -> None:
    leaves, fn = case
    want = torch.autograd.grad(fn(*leaves), leaves)
    torch._dynamo.reset()
    got = torch.autograd.grad(torch.compile(fn, backend="aot_eager")(*leaves), leaves)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_upstream_gradients_that_stand_for_their_negatives() -> None:
    announce("row operators negated upstream gradients")
    up = torch.view_as_complex(torch.randn(60, 40, 2, device=DEV)).conj().imag
    assert up.is_neg()
    x = torch.randn(60, 40, device=DEV, requires_grad=True)
    w = torch.randn(40, 40, device=DEV)
    for y in (layer_norm_hip(x), gated_linear_hip(x, w, w)):
        a, b = torch.autograd.grad(y, x, up, retain_graph=True)[0], torch.autograd.grad(y, x, up.clone())[0]
        assert torch.equal(a, b)


def test_calls_from_two_threads_on_two_streams() -> None:
    announce("row operators from two threads")
    wrong: list[str] = []

    def work(seed: int) -> None:
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                made = [make(seed=seed) for make in CASES.values()]
                stream.synchronize()
                first = None
                for _ in range(20):
                    now = [g for leaves, fn in made for g in torch.autograd.grad(fn(*leaves), leaves)]
                    stream.synchronize()
                    if first is None:
                        first = [t.clone() for t in now]
                    elif not all(torch.equal(a, b) for a, b in zip(first, now)):
                        wrong.append(f"thread {seed}")
                        return
        except Exception as exc:  # noqa: BLE001 (reported by the test)
            wrong.append(repr(exc))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


# What comes back instead of the n-th saved tensor.
OTHERS = {
    "on the CPU": lambda t: t.cpu(),
    "a row less": lambda t: t[..., :-1] if t.dim() else t.cpu(),
    "of another type": lambda t: t.double() if t.is_floating_point() else t.int(),
    "of another order": lambda t: t.reshape(-1),
}


@pytest.mark.parametrize("other", OTHERS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("name", ["lnorm", "gated", "distill"])
def test_others_are_refused(name, dtype, other) -> None:
    leaves, fn = CASES[name](dtype)
    count = [0]

    def pack(t):
        count[0] += 1
        return count[0] - 1, t

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda held: held[1]):
        torch.autograd.grad(fn(*leaves), leaves)
    saved = count[0]
    refused = 0
    for n in range(saved):
        announce(f"hooks {name} {dtype}: saved tensor {n} {other}")
        count[0] = 0

        def unpack(held):
            return OTHERS[other](held[1]) if held[0] == n else held[1]

        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            loss = fn(*leaves)
        try:
            torch.autograd.grad(loss, leaves)
        except (ValueError, RuntimeError):
            refused += 1
    # "of another order" leaves vectors as they are; what other operations of the case save is theirs
    assert refused == saved if other != "of another order" else refused >= 1
