"""Norms and loss where the module of native calls is missing (``-m gpu``): the operators give the same numbers."""

from __future__ import annotations

import sys

import pytest
import torch

from omniwave_amd import AdamW, _native, block_norms_hip, cross_entropy_hip, rms_norm_hip

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def announce(msg: str) -> None:
    print(f"\n[gpu-case] {msg}", file=sys.stderr, flush=True)


def results(dtype):
    gen = torch.Generator(device=DEV).manual_seed(3)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=DEV).to(dtype).requires_grad_(True)

    x, delta, w, gate, nxt = normal(3, 50, 95), normal(3, 50, 95), normal(95), normal(3, 95), normal(95)
    out = block_norms_hip(x, delta, post_weight=w, gate=gate, next_weight=nxt)
    found = [*out, *torch.autograd.grad(out, (x, delta, w, gate, nxt), [torch.ones_like(o) for o in out])]
    y = rms_norm_hip(x, w)
    found += [y, *torch.autograd.grad(y, (x, w), torch.ones_like(y))]
    logits, a = normal(40, 1000), torch.randint(0, 1000, (40,), generator=gen, device=DEV)
    for reduction in ("mean", "sum"):
        loss = cross_entropy_hip(logits, a, target_b=a.flip(0), mix=0.3, label_smoothing=0.1, reduction=reduction)
        found += [loss, *torch.autograd.grad(loss, logits)]
    return [t.detach() for t in found]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_operators_alone(dtype, monkeypatch) -> None:
    announce(f"norms and loss without native calls {dtype}")
    want = results(dtype)
    monkeypatch.setattr(_native, "_glue", None)
    monkeypatch.setattr(_native, "_glue_error", "cannot load _glue.so")
    found = results(dtype)
    assert all(a.dtype == b.dtype and torch.equal(a, b) for a, b in zip(want, found))
    p = torch.nn.Parameter(torch.ones(5, device=DEV))
    p.grad = torch.ones_like(p)
    with pytest.raises(RuntimeError, match="_glue.so"):
        AdamW([p]).step()
