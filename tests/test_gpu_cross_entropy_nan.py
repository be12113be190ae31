"""A NaN among a row's logits is in its loss and in its whole gradient, wherever it lies (``-m gpu``): in a
thread's only value, among masked classes (-inf), in short and long rows, in few and many of them.

By the definition log z and every probability of such a row are NaN and the other rows are what they are
without it, so nothing here has a tolerance.
"""

from __future__ import annotations

import sys

import pytest
import torch

from omniwave_amd import cross_entropy_hip

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
NAN, INF = float("nan"), float("inf")


def announce(msg: str) -> None:
    print(f"\n[gpu-case] {msg}", file=sys.stderr, flush=True)


def run(x, target, reduction):
    x = x.to(DEV).requires_grad_(True)
    loss = cross_entropy_hip(x, target.to(DEV), reduction=reduction)
    (grad,) = torch.autograd.grad(loss.sum(), x)
    return loss.detach().cpu(), grad.cpu()


def make(rows, k, at, dtype, masked):
    """Rows of logits with their labels beside class ``at[row]``, which is to be NaN; ``masked``: every other
    class but the label is -inf."""
    gen = torch.Generator().manual_seed(rows + k)
    x = torch.randn(rows, k, generator=gen)
    target = (at + 1) % k
    if masked:
        picked = x.gather(1, target[:, None])
        x = torch.full_like(x, -INF).scatter_(1, target[:, None], picked)
    return x.to(dtype), target


def check(rows, k, at, dtype, masked):
    """Every second row has its NaN."""
    x, target = make(rows, k, at, dtype, masked)
    bad = torch.arange(rows) % 2 == 0
    poisoned = torch.where(bad[:, None] & (torch.arange(k) == at[:, None]), NAN, x.float()).to(dtype)
    clean_loss, clean_grad = run(x, target, "none")
    loss, grad = run(poisoned, target, "none")
    assert loss[bad].isnan().all() and torch.equal(loss[~bad], clean_loss[~bad])
    assert grad[bad].isnan().all() and torch.equal(grad[~bad], clean_grad[~bad])
    for reduction in ("sum", "mean"):
        loss, grad = run(poisoned, target, reduction)
        assert loss.isnan() and grad[bad].isnan().all() and grad[~bad].isfinite().all()
        # A row that is left out has nothing of its NaN.
        loss, grad = run(poisoned, torch.where(bad, -100, target), reduction)
        assert not grad[bad].any()
        assert grad[~bad].isfinite().all() and (loss.isfinite() or (reduction == "mean" and bad.all()))


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("k", [2, 3, 7, 10, 11, 23, 63])
def test_every_class_of_short_rows(k, dtype, masked) -> None:
    announce(f"xent nan k={k} {dtype} masked={masked}")
    for at in range(k):
        check(2, k, torch.full((2,), at), TYPES[dtype], masked)  # a workgroup, a wave a row
    check(2 * k, k, torch.arange(2 * k) // 2, TYPES[dtype], masked)


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,k", [(2, 1000), (300, 1000), (2500, 1000), (2300, 4000), (9, 4097), (300, 5003), (4, 20000),
                                    (3, 20005), (5000, 3), (9001, 7), (9001, 10), (20000, 23), (9001, 100)])
def test_few_and_many_rows(rows, k, dtype, masked) -> None:
    announce(f"xent nan rows={rows} k={k} {dtype} masked={masked}")
    at = torch.randint(0, k, (rows,), generator=torch.Generator().manual_seed(rows))
    at[:4] = torch.tensor([k - 1, k - 1, 0, 0])[:rows]
    check(rows, k, at, TYPES[dtype], masked)


@pytest.mark.parametrize("k", [2, 10, 1000, 20003])
def test_rows_of_nan_alone(k) -> None:
    announce(f"xent rows of nan k={k}")
    x, target = torch.full((3, k), NAN), torch.zeros(3, dtype=torch.int64)
    x[1, 0] = 0.5  # but for the label
    x[2] = 0.25
    loss, grad = run(x, target, "none")
    assert loss[:2].isnan().all() and grad[:2].isnan().all() and loss[2].isfinite() and grad[2].isfinite().all()
