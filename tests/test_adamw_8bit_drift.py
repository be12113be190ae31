"""How far the 8-bit root of the second moment strays from the 32-bit one over thousands of steps (the format alone, on
the CPU): the limits that ``AdamW`` documents.

The root is rounded to the nearest code after each step, and a step moves it by 0.05% (beta2 = 0.999), where half a
step between codes is 3 to 6%.  What a block of 256 has in common is followed by its scale, which is fp32.  A value's
part of the block's largest one moves only by gradients that change it by half a code's step at once:
* it never falls by less, so after gradients fall tenfold beside a steady one the root is at most the fall times
  what it strayed before;
* a rise by the factor f reaches at least 1 / f of the right root, times what it strayed before.
Where nothing changes the root strays by the codes that large gradients left, between half and twice the right one.
"""

from __future__ import annotations

import pytest
import torch

from omniwave_amd.optim import BLOCK, _decode, _encode

BLOCKS, STEPS, CHANGE, BETA2 = 32, 3000, 500, 0.999
STRAY = (0.5, 2.5)  # of nearly all values where nothing changes


def ratios(factor: float, steady: bool) -> torch.Tensor:
    """8-bit roots over 32-bit ones after STEPS steps; gradients change by ``factor`` after CHANGE of them, but for one
    of each block where ``steady``."""
    gen = torch.Generator().manual_seed(0)
    n = BLOCKS * BLOCK
    size = torch.exp(0.7 * torch.randn(n, generator=gen)).view(BLOCKS, BLOCK)
    if steady:
        size[:, 0] = 9.0
    size = size.view(-1)
    later = (size * factor).view(BLOCKS, BLOCK)
    if steady:
        later[:, 0] = 9.0
    codes, scale = _encode(torch.zeros(n), True)
    v = torch.zeros(n)
    for t in range(STEPS):
        g = (size if t < CHANGE else later.view(-1)) * torch.randn(n, generator=gen)
        codes, scale = _encode((_decode(codes, scale).square() * BETA2 + g * g * (1 - BETA2)).sqrt(), True)
        v = v * BETA2 + g * g * (1 - BETA2)
    return (_decode(codes, scale) / v.sqrt()).view(BLOCKS, BLOCK)[:, 1:].reshape(-1)


def inside(r: torch.Tensor, low: float, high: float) -> None:
    """Nearly all ratios (1% to 99%) between two bounds."""
    found = torch.quantile(r, torch.tensor([0.01, 0.99])).tolist()
    assert low <= found[0] and found[1] <= high, found


@pytest.mark.parametrize("factor", [1.0, 0.1, 4.0])
def test_what_a_block_has_in_common_is_followed(factor) -> None:
    r = ratios(factor, steady=False)
    inside(r, *STRAY)
    assert 0.9 <= r.median().item() <= 1.1


def test_a_fall_beside_a_steady_value_is_not_followed() -> None:
    r = ratios(0.1, steady=True)
    inside(r, STRAY[0], 10 * STRAY[1])
    assert r.median().item() > 2  # the documented limit, not a wish: a format that follows may say so


def test_a_rise_beside_a_steady_value_is_followed_in_part() -> None:
    inside(ratios(4.0, steady=True), STRAY[0] / 4, STRAY[1])
