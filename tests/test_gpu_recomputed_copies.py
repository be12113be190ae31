"""Operators called with tensors that have to be copied first (``-m gpu``), which go through ``torch.library``, under recomputation and hooks
on saved tensors: each saved tensor is asked for once."""

from __future__ import annotations

import sys

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from omniwave_amd import (block_norms_hip, cross_entropy_hip, distillation_hip, gated_linear_hip, layer_norm_hip,
                          rms_norm_hip)

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def announce(msg: str) -> None:
    print(f"\n[gpu-case] {msg}", file=sys.stderr, flush=True)


def make(name):
    """(leaves, a function of them): every tensor of rows lies across its memory."""
    gen = torch.Generator().manual_seed(0)
    normal = lambda *shape: torch.randn(shape, generator=gen).to(DEV)
    x, delta = normal(3, 24, 5, 5).permute(0, 2, 3, 1), normal(3, 24, 5, 5).permute(0, 2, 3, 1)
    w, b, wide = normal(24), normal(24), normal(24, 16).T
    labels = torch.randint(0, 24, (3, 5, 5), generator=gen).to(DEV)
    values, classes = normal(3, 5, 5, 24).topk(4, -1)
    return {
        "layer norm": ([x, w, b], lambda x, w, b: layer_norm_hip(x, w, b)),
        "layer norm without bias": ([x, w], lambda x, w: layer_norm_hip(x, w)),
        "rms norm": ([x, w], rms_norm_hip),
        "block norms": ([x, delta, w, b], lambda x, d, w, b: block_norms_hip(x, d, post_weight=w, gate=b)[0]),
        "gated": ([x, wide, wide.clone()], gated_linear_hip),
        "cross-entropy": ([x], lambda x: cross_entropy_hip(x.reshape(75, 24).T.contiguous().T, labels.reshape(-1), reduction="none")),
        "distillation": ([x], lambda x: distillation_hip(x, values, classes, reduction="none")),
    }[name]


NAMES = ["layer norm", "layer norm without bias", "rms norm", "block norms", "gated", "cross-entropy", "distillation"]


@pytest.mark.parametrize("name", NAMES)
def test_recomputation(name) -> None:
    announce(f"recomputation of {name} with copies")
    leaves, fn = make(name)
    leaves = [t.detach().requires_grad_(True) for t in leaves]
    out = fn(*leaves)
    up = torch.randn(out.shape, generator=torch.Generator().manual_seed(1)).to(DEV)
    want = torch.autograd.grad(out, leaves, up)
    again = checkpoint(fn, *leaves, use_reentrant=False)
    assert torch.equal(again, out) and all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(again, leaves, up), want))


@pytest.mark.parametrize("name", NAMES)
def test_hooks_run_once(name) -> None:
    announce(f"hooks on saved tensors of {name} with copies")
    leaves, fn = make(name)
    leaves = [t.detach().requires_grad_(True) for t in leaves]
    packed, unpacked = [], []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: packed.append(t) or len(packed) - 1,
                                                  lambda n: unpacked.append(n) or packed[n]):
        out = fn(*leaves)
    out.sum().backward()
    assert sorted(unpacked) == list(range(len(packed)))
