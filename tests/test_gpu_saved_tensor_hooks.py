"""Hooks on saved tensors that hand out others than were saved (``-m gpu``): the backward of norms and loss says so before
anything is launched; copies that lie otherwise are taken."""

from __future__ import annotations

import sys

import pytest
import torch

from omniwave_amd import block_norms_hip, cross_entropy_hip, rms_norm_hip

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def announce(msg: str) -> None:
    print(f"\n[gpu-case] {msg}", file=sys.stderr, flush=True)


def norms(dtype):
    x, delta = (torch.randn(2, 30, 96, device=DEV).to(dtype).requires_grad_(True) for _ in range(2))
    w = [torch.rand(96, device=DEV).requires_grad_(True) for _ in range(3)]
    return [x, delta, *w], lambda: sum(t.float().sum() for t in block_norms_hip(
        x, delta, post_weight=w[0], gate=w[1], scale=torch.ones(2, device=DEV), next_weight=w[2]))


def rms(dtype):
    x, w = torch.randn(2, 30, 96, device=DEV).to(dtype).requires_grad_(True), torch.rand(96, device=DEV).requires_grad_(True)
    return [x, w], lambda: rms_norm_hip(x, w).float().sum()


def xent(dtype):
    x = torch.randn(20, 96, device=DEV).to(dtype).requires_grad_(True)
    a, b = (torch.randint(0, 96, (20,), device=DEV) for _ in range(2))
    return [x], lambda: cross_entropy_hip(x, a, target_b=b, mix=torch.rand(20, device=DEV))


# What comes back instead of the n-th saved tensor.
OTHERS = {
    "on the CPU": lambda t: t.cpu(),
    "a row less": lambda t: t[..., :-1] if t.dim() else t.cpu(),
    "of another type": lambda t: t.double() if t.is_floating_point() else t.int(),
    "of another order": lambda t: t.reshape(-1),
}


@pytest.mark.parametrize("other", OTHERS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("make", [norms, rms, xent])
def test_others_are_refused(make, dtype, other) -> None:
    leaves, call = make(dtype)
    count = [0]

    def pack(t):
        count[0] += 1
        return count[0] - 1, t

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda held: held[1]):
        torch.autograd.grad(call(), leaves)
    saved = count[0]
    assert saved >= 2
    refused = 0
    for n in range(saved):
        announce(f"hooks {make.__name__} {dtype}: saved tensor {n} {other}")
        count[0] = 0

        def unpack(held):
            return OTHERS[other](held[1]) if held[0] == n else held[1]

        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            loss = call()
        try:
            torch.autograd.grad(loss, leaves)
        except (ValueError, RuntimeError):
            refused += 1
    # "of another order" leaves vectors as they are
    assert refused == saved if other != "of another order" else refused >= 1


@pytest.mark.parametrize("make", [norms, rms, xent])
def test_copies_that_lie_otherwise_are_taken(make) -> None:
    announce(f"hooks {make.__name__}: strided copies")
    torch.manual_seed(0)
    leaves, call = make(torch.float32)
    torch.manual_seed(1)
    want = torch.autograd.grad(call(), leaves)

    def strided(t):
        return t if t.dim() == 0 else torch.stack([t, t], -1)[..., 0]

    torch.manual_seed(1)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, strided):
        loss = call()
        got = torch.autograd.grad(loss, leaves)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("make", [norms, rms, xent])
def test_upstream_gradients_that_stand_for_their_negatives(make) -> None:
    announce(f"negated upstream gradients {make.__name__}")
    leaves, call = make(torch.float32)
    torch.manual_seed(1)
    loss = call()
    want = torch.autograd.grad(loss, leaves, torch.full((), 2.0, device=DEV), retain_graph=True)
    up = torch._neg_view(torch.full((), -2.0, device=DEV))  # as the imaginary part of a conjugate is one
    assert up.is_neg() and up.item() == 2.0
    got = torch.autograd.grad(loss, leaves, up)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_upstream_gradients_of_outputs_that_stand_for_their_negatives() -> None:
    announce("negated upstream gradients of the norms' outputs")
    x, delta = (torch.randn(2, 30, 96, device=DEV, requires_grad=True) for _ in range(2))
    w, up = torch.rand(96, device=DEV), torch.randn(2, 30, 96, device=DEV)
    out = block_norms_hip(x, delta, next_weight=w)
    want = torch.autograd.grad(out, (x, delta), (up, up), retain_graph=True)
    got = torch.autograd.grad(out, (x, delta), (torch._neg_view(-up), torch._neg_view(-up)))
    assert all(torch.equal(a, b) for a, b in zip(want, got))
