"""The registered operators behind norms and loss check what they are given themselves, before an address goes to a kernel:
they can be called by their names, and a backward gets what hooks on saved tensors hand out (on the CPU, with the launch
replaced by a record)."""

from __future__ import annotations

import pytest
import torch

from omniwave_amd import loss, norms


@pytest.fixture
def launches(monkeypatch):
    calls = []
    for module in (norms, loss):
        monkeypatch.setattr(module, "_on", lambda *args: calls.append(args))
        monkeypatch.setattr(module, "gpu_reason", lambda t: None)
    class Anywhere:
        def __init__(self, device):
            pass

        def __enter__(self):
            pass

        def __exit__(self, *args):
            pass

    monkeypatch.setattr(torch.cuda, "device", Anywhere)
    return calls


def norm_tensors(**other):
    t = dict(x=torch.zeros(2, 5, 24), delta=torch.zeros(2, 5, 24), post_weight=torch.ones(24), gate=torch.ones(2, 24),
             scale=torch.ones(2), next_weight=torch.ones(24))
    return {**t, **other}


BAD_NORMS = {
    "delta of another type": dict(delta=torch.zeros(2, 5, 24).bfloat16()),
    "delta of another shape": dict(delta=torch.zeros(2, 4, 24)),
    "a short weight": dict(post_weight=torch.ones(23)),
    "a short gate": dict(gate=torch.ones(1, 24)),
    "a short scale": dict(scale=torch.ones(1)),
    "a weight of integers": dict(next_weight=torch.ones(24, dtype=torch.int32)),
    "x of doubles": dict(x=torch.zeros(2, 5, 24).double(), delta=torch.zeros(2, 5, 24).double()),
    "elsewhere": dict(delta=torch.zeros(2, 5, 24, device="meta")),
}


@pytest.mark.parametrize("bad", BAD_NORMS)
def test_norms(launches, bad) -> None:
    t = norm_tensors(**BAD_NORMS[bad])
    with pytest.raises(ValueError):
        norms._run_forward(*t.values(), 1e-6)
    up = torch.zeros(2, 5, 24, dtype=t["x"].dtype)
    with pytest.raises(ValueError):
        norms._run_backward(up, up, *t.values(), 1e-6, [True] * 5)
    assert not launches


@pytest.mark.parametrize("up", [torch.zeros(2, 5, 23), torch.zeros(2, 5, 24).bfloat16(), torch.zeros(10, 24),
                                torch.zeros(2, 5, 24, device="meta")])
def test_upstream_gradients_of_norms(launches, up) -> None:
    t, good = norm_tensors(), torch.zeros(2, 5, 24)
    for dout, dnext in ((up, good), (good, up), (up, None), (None, up)):
        with pytest.raises(ValueError, match="upstream"):
            norms._run_backward(dout, dnext, *t.values(), 1e-6, [True] * 5)
    assert not launches
    norms._run_backward(good, good, *t.values(), 1e-6, [True] * 5)
    norms._run_forward(*t.values(), 1e-6)
    assert len(launches) == 2


def loss_tensors(**other):
    t = dict(logits=torch.zeros(6, 10), target=torch.zeros(6, dtype=torch.int64), target_b=torch.zeros(6, dtype=torch.int64),
             mix=torch.ones(6))
    return {**t, **other}


BAD_LOSS = {
    "doubles": dict(logits=torch.zeros(6, 10).double()),
    "fewer labels": dict(target=torch.zeros(5, dtype=torch.int64)),
    "labels of 32 bits": dict(target=torch.zeros(6, dtype=torch.int32)),
    "fewer second labels": dict(target_b=torch.zeros(5, dtype=torch.int64)),
    "fewer weights": dict(mix=torch.ones(5)),
    "labels elsewhere": dict(target=torch.zeros(6, dtype=torch.int64, device="meta")),
}
OPTIONS = (1.0, 0.1, -100, 2)


@pytest.mark.parametrize("bad", BAD_LOSS)
def test_loss(launches, bad) -> None:
    t = loss_tensors(**BAD_LOSS[bad])
    with pytest.raises(ValueError):
        loss._run_forward(*t.values(), *OPTIONS)
    with pytest.raises(ValueError):
        loss._run_backward(torch.ones(()), torch.zeros(19), *t.values(), *OPTIONS)
    assert not launches


def test_what_the_backward_of_the_loss_gets(launches) -> None:
    t = loss_tensors()
    for up, aux in ((torch.ones(2), torch.zeros(19)), (torch.ones(()), torch.zeros(18)), (torch.ones(()), torch.zeros(19).half()),
                    (torch.ones((), device="meta"), torch.zeros(19)), (torch.ones(()), torch.zeros(19, device="meta"))):
        with pytest.raises(ValueError, match="backward"):
            loss._run_backward(up, aux, *t.values(), *OPTIONS)
    with pytest.raises(ValueError, match="backward"):
        loss._run_backward(torch.ones(()), torch.zeros(13), *t.values(), 1.0, 0.1, -100, 0)  # a gradient for each row
    assert not launches
    loss._run_backward(torch.ones(()), torch.zeros(19), *t.values(), *OPTIONS)
    loss._run_backward(torch.ones(6), torch.zeros(13), *t.values(), 1.0, 0.1, -100, 0)
    assert len(launches) == 2


def test_the_device_is_looked_at() -> None:
    t, u = norm_tensors(), loss_tensors()
    ops = torch.ops.omniwave_amd
    up = torch.zeros(2, 5, 24)
    for call in (lambda: ops.block_norms_fwd(*t.values(), 1e-6), lambda: ops.cross_entropy_fwd(*u.values(), *OPTIONS),
                 lambda: ops.block_norms_bwd(up, up, *t.values(), 1e-6, [True] * 5),
                 lambda: ops.cross_entropy_bwd(torch.ones(()), torch.zeros(19), *u.values(), *OPTIONS)):
        with pytest.raises(RuntimeError, match="not supported"):
            call()
