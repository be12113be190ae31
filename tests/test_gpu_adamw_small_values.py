"""AdamW with gradients whose squares are subnormal (``-m gpu``): the root of the second moment is what the
formula says, which a step shows where eps does not hide it."""

from __future__ import annotations

import sys

import pytest
import torch

from omniwave_amd import AdamW

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
U = 2.0 ** -24


def announce(msg: str) -> None:
    print(f"\n[gpu-case] {msg}", file=sys.stderr, flush=True)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps", [0.0, 1e-30])
def test_subnormal_second_moments(bits, eps) -> None:
    announce(f"adamw subnormal squares bits={bits} eps={eps}")
    # Squares from 1e-34 down to 2e-40, times 1e-3: 400 least steps of fp32 at the end.
    n = 5000
    g = torch.logspace(-17, -19.7, n, dtype=torch.float64).float() * torch.where(torch.arange(n) % 3 == 0, -1.0, 1.0)
    p = torch.nn.Parameter(torch.zeros(n, device=DEV))
    p.grad = g.to(DEV)
    lr, b1, b2 = 1e-3, 0.9, 0.999
    AdamW([p], lr=lr, betas=(b1, b2), eps=eps, weight_decay=0.0, state_bits=bits).step()
    g = g.double()
    m, v = (1 - b1) * g, (1 - b2) * g * g
    want = -lr * (m / (1 - b1)) / ((v / (1 - b2)).sqrt() + eps)
    # v: three roundings, each of at most half a least step (2^-150) or U, halved by the root; the others are ten
    # roundings, and two units each for 1 - b (0.1 and 0.001 as fp32 numbers), the quotient and expm1.
    slack = want.abs() * (0.75 * 2.0 ** -149 / v + 30 * U)
    gap = (p.detach().cpu().double() - want).abs() - slack
    assert gap.max().item() <= 0, f"{gap.max().item()} past the bound"
