"""The native calls' autograd nodes on the GPU (``-m gpu``): hooks, recomputation, a second derivative, calls at
once, compilation, and that the plain case takes them."""

from __future__ import annotations

import sys
import threading

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from omniwave_amd import _native, block_norms_hip, cross_entropy_hip, rms_norm_hip

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def announce(msg: str) -> None:
    print(f"\n[gpu-case] {msg}", file=sys.stderr, flush=True)


def norms_inputs(seed=0, rows=49, c=256):
    gen = torch.Generator().manual_seed(seed)
    t = [torch.randn(2, rows, c, generator=gen).bfloat16().to(DEV).requires_grad_(True) for _ in range(2)]
    w = [(torch.rand(c, generator=gen) + 0.5).to(DEV).requires_grad_(True) for _ in range(3)]
    return [*t, *w]


def norms_loss(x, delta, post, gate, nxt):
    out, n = block_norms_hip(x, delta, post_weight=post, gate=gate, next_weight=nxt)
    return (out.float() * 0.5).sum() + (n.float() * 2).sum()


def xent_inputs(seed=0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(33, 1000, generator=gen).to(DEV).requires_grad_(True)
    return [x], torch.randint(0, 1000, (33,), generator=gen).to(DEV)


CASES = {"norms": lambda: (norms_inputs(), norms_loss), "rms": lambda: (norms_inputs()[::4], lambda x, w: rms_norm_hip(x, w).float().sum())}


def _xent_case():
    leaves, labels = xent_inputs()
    return leaves, lambda x: cross_entropy_hip(x, labels, label_smoothing=0.1)


CASES["xent"] = _xent_case


@pytest.fixture(params=sorted(CASES))
def case(request):
    announce(f"native call {request.param}")
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
    assert calls and all(calls)


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


def test_calls_from_two_threads_on_two_streams() -> None:
    announce("native calls from two threads")
    wrong: list[str] = []

    def work(seed: int) -> None:
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                leaves = norms_inputs(seed)
                rows, labels = xent_inputs(seed)
                stream.synchronize()
                first = None
                for _ in range(20):
                    now = [*torch.autograd.grad(norms_loss(*leaves), leaves),
                           *torch.autograd.grad(cross_entropy_hip(rows[0], labels), rows)]
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
