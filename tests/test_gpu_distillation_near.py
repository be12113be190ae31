"""Distillation from lists of all classes on the GPU (``-m gpu``), where the student is near its teacher: the loss is a small rest
of sums that cancel, and keeps its digits.  Against the formula in 64 bits.

Tolerances, in half steps U = 2^-24 of fp32.  With d = ln(p / q) a row's loss is T^2 sum q (e^d - 1 - d).  A sum of exponentials is
within (4 |x - m| / T + 420) U of itself, its terms weighed by what they are; ln of the quotient of two such sums is off by D, the
error of both and of the logarithm.  D is common to all entries and sum q (e^d - 1) = 0, so it enters as D^2 / 2 (a little more, for
the second term of the series is e^d / 2).  Each d is off by 4 U (|d| + ln of the quotient) besides, which enters times q |e^d - 1|;
q by (4 |t - mt| / T + 430) U of itself, the polynomial, the sum over at most 1,024 terms a lane and the last products by (top / 16 +
100) U of the loss.  Losses from T^2 / 32 on are formed from the logarithms and have their error instead: 900 U, 4 U of each logarithm, and for
each entry its share of 4 |t - mt| / T + 900 U of the magnitudes of both differences.  Where |d| >= 1/2 the terms are p - q - q d, of exponentials one by one: (4 |x - m| / T + 900) U p and (4 |t - mt| / T +
440) U q (1 + |d|).
"""

from __future__ import annotations

import sys

import pytest
import torch

from omniwave_amd import distillation_hip

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
U = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def announce(msg: str) -> None:
    print(f"\n[gpu-case] {msg}", file=sys.stderr, flush=True)


def formula(x, v, i, temp):
    """(losses, their allowance) of lists of all classes."""
    x, t = x.double().gather(1, i) / temp, v.double() / temp
    dx, dt = x - x.amax(1, keepdim=True), t - t.amax(1, keepdim=True)
    log_z, log_zt = dx.logsumexp(1, keepdim=True), dt.logsumexp(1, keepdim=True)
    p, q = (dx - log_z).exp(), (dt - log_zt).exp()
    ratio = log_z - log_zt
    d = dx - dt - ratio
    losses = -(q * d).sum(1)
    off = U * (4 * (p * dx.abs()).sum(1) + 4 * (q * dt.abs()).sum(1) + 850 + ratio.abs()[:, 0])
    far = d.abs() >= 0.49
    each = (q * d.expm1().abs() * 4 * U * (d.abs() + ratio.abs())).sum(1)
    near = torch.where(far, 0, q * (d.expm1() - d) * (4 * dt.abs() + 430) * U).sum(1)
    gone = torch.where(far, p * (4 * dx.abs() + 900) * U + q * (1 + d.abs()) * (4 * dt.abs() + 440) * U, 0).sum(1)
    slack = 0.6 * off ** 2 + each + near + gone + (v.shape[1] / 16 + 100) * U * losses.abs()
    plain = 900 + 4 * (log_z + log_zt)[:, 0] + (q * (4 * dt.abs() + 900) * (dt.abs() + torch.where(q > 0, dx.abs(), 0))).sum(1)
    slack = torch.where(losses < 0.031, slack, slack + U * plain)
    return temp ** 2 * losses, temp ** 2 * slack


def make(rows, k, noise, dtype, shift=0.0, scale=2.0):
    gen = torch.Generator().manual_seed(rows + k)
    teacher = torch.randn(rows, k, generator=gen) * scale
    x = (teacher + shift + torch.randn(rows, k, generator=gen) * noise).to(dtype)
    i = torch.stack([torch.randperm(k, generator=gen) for _ in range(rows)])
    return x.to(DEV), teacher.gather(1, i).to(DEV), i.to(DEV)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("temp", [1.0, 4.0, 0.5])
@pytest.mark.parametrize("rows,k", [(1, 2), (8, 10), (8, 1000), (40, 1000), (5, 5000), (2, 20000), (2100, 30), (2100, 100),
                                    (2100, 300), (2100, 700), (9000, 21)])
def test_near_students(rows, k, temp, dtype) -> None:
    announce(f"distillation near its teacher rows={rows} k={k} T={temp} {dtype}")
    for noise in (0.01, 0.1, 1.0):
        x, v, i = make(rows, k, noise, TYPES[dtype])
        ref, slack = formula(x, v, i, temp)
        losses = distillation_hip(x, v, i, temperature=temp, reduction="none")
        gap = ((losses.double() - ref).abs() - slack).max().item()
        assert gap <= 0, f"noise {noise}: {gap} past the bound"
        # The bound is a small part of the losses: D is below 2,000 U, its square 1.4e-8 T^2, while a loss is about noise^2 / 2 of the
        # share that the largest class leaves, 5e-5 of it for 0.01.  A row whose one class has nearly everything may have less
        # than its bound, their mean has not.
        if k >= 100:
            assert slack.mean() <= 0.01 * ref.mean()
        mean = distillation_hip(x, v, i, temperature=temp)
        assert abs(mean.item() - ref.mean().item()) <= slack.mean().item() + 4 * U * ref.mean().item()


@pytest.mark.parametrize("temp", [1.0, 4.0, 20.0])
@pytest.mark.parametrize("k", [10, 1000, 20000])
def test_the_nearer_the_smaller(k, temp) -> None:
    announce(f"distillation ever nearer to its teacher k={k} T={temp}")
    for noise in (1e-3, 1e-4, 0.0):
        x, v, i = make(6, k, noise, torch.float32)
        ref, slack = formula(x, v, i, temp)
        losses = distillation_hip(x, v, i, temperature=temp, reduction="none")
        assert (losses >= 0).all() and ((losses.double() - ref).abs() <= slack).all()


def test_logits_of_another_height() -> None:
    announce("distillation near its teacher, 1,000 above it")
    x, v, i = make(7, 300, 0.05, torch.float32, shift=1000.0)
    ref, slack = formula(x, v, i, 2.0)
    losses = distillation_hip(x, v, i, temperature=2.0, reduction="none")
    assert ((losses.double() - ref).abs() <= slack).all() and (slack <= 0.01 * ref).all()


def test_classes_that_the_teacher_all_but_rules_out() -> None:
    """Entries whose q is 0 in fp32 bring the student's share of their classes."""
    announce("distillation of classes without a share")
    x, v, i = make(5, 50, 0.01, torch.float32)
    v[:, 3:9] = -400.0
    ref, slack = formula(x, v, i, 1.0)
    losses = distillation_hip(x, v, i, reduction="none")
    assert ((losses.double() - ref).abs() <= slack).all()
    x.scatter_(1, i[:, 5:7], -float("inf"))  # the student, too
    losses = distillation_hip(x, v, i, reduction="none")
    assert losses.isfinite().all() and (losses > 0).all()
    x.scatter_(1, i[:, :1], -float("inf"))  # what the teacher wants
    assert (distillation_hip(x, v, i, reduction="none") == float("inf")).all()


def test_lists_as_long_as_the_classes_that_miss_some() -> None:
    """As many entries as classes, one class twice and one never; then one entry that is none.  The loss is the definition's, within
    its sums' rounding and, where the two classes have nearly the same share, the (128 + classes / 16) U at which such a
    list is taken for whole."""
    announce("distillation of lists that are not whole")
    k, temp = 300, 2.0
    x, v, i = make(6, k, 0.01, torch.float32)
    i[:, 1] = i[:, 0]
    x[3] = 0.0
    log_p, t = (x.double() / temp).log_softmax(1), v.double() / temp
    ref = temp ** 2 * (t.softmax(1) * (t.log_softmax(1) - log_p.gather(1, i))).sum(1)
    slack = temp ** 2 * U * (1800 + 4 * k + 8 * (t.softmax(1) * (t.abs() + log_p.gather(1, i).abs()) ** 2).sum(1))
    losses = distillation_hip(x, v, i, temperature=temp, reduction="none")
    assert ((losses.double() - ref).abs() <= slack).all()
    x, v, i = make(6, k, 0.01, torch.float32)
    v[:, 4] = -float("inf")
    log_p, t = (x.double() / temp).log_softmax(1), v.double() / temp
    q = t.softmax(1)
    ref = temp ** 2 * torch.where(q > 0, q * (t.log_softmax(1) - log_p.gather(1, i)), 0).sum(1)
    losses = distillation_hip(x, v, i, temperature=temp, reduction="none")
    assert ((losses.double() - ref).abs() <= slack).all()


@pytest.mark.parametrize("rows,k,top", [(3, 10, 25), (3, 300, 301), (2, 17000, 17500), (2100, 40, 64)])
def test_lists_longer_than_the_classes(rows, k, top) -> None:
    """All classes among entries that are none, of an ignored class and of logits that are no numbers there: the loss of the classes."""
    announce(f"distillation of {k} classes among {top} entries")
    x, v, i = make(rows, k, 0.01, torch.float32)
    ref, slack = formula(x, v, i, 2.0)
    gen = torch.Generator().manual_seed(5)
    for ignore in (-100, 1 << 40):
        at = torch.stack([torch.randperm(top, generator=gen)[:k] for _ in range(rows)]).to(DEV)
        classes = torch.full((rows, top), ignore, device=DEV).scatter_(1, at, i)
        values = torch.full((rows, top), float("nan"), device=DEV).scatter_(1, at, v)
        losses = distillation_hip(x, values, classes, temperature=2.0, ignore_index=ignore, reduction="none")
        assert ((losses.double() - ref).abs() <= slack + 600 * U * ref).all()  # the lanes' sums are in another order
