"""Gated feed-forward product on the GPU (``-m gpu``) where G and U are so large that their product leaves fp32's range, and
the gate closes: silu(G) U, and both gradients, are 0 there (e^-1e20 is), and everything else is as if these tokens were zeros.

No tolerances: the tokens' exact results are 0, and a token of zeros has h = 0, dU = dh silu(0) = 0 and dG = dh U f = 0 (U = 0),
so all other results and the weights' gradients are the same sums of the same values.
"""

from __future__ import annotations

import sys

import pytest
import torch

from omniwave_amd import gated_linear_hip

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def announce(msg: str) -> None:
    print(f"\n[gpu-case] {msg}", file=sys.stderr, flush=True)


def run(x, wg, wu, dh):
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, wg, wu)]
    with torch.no_grad():
        plain = gated_linear_hip(x, wg, wu)  # a call without a graph keeps no products
    h = gated_linear_hip(*leaves)
    assert torch.equal(h.detach(), plain)
    return h.detach(), *torch.autograd.grad(h, leaves, dh)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,c,hidden", [
    (5, 64, 40),        # few tokens, products formed again in the backward
    (40, 1536, 24),     # the same, kept (16 bits)
    (60, 200, 40),      # the same, kept (fp32)
    (6000, 64, 96),     # tiles
    (300, 1408, 130),   # parts of tiles, joined
    (300, 2064, 70),    # the same, kept
    (6000, 2048, 64),   # tiles, kept
])
def test_closed_gates_of_large_products(rows, c, hidden, dtype) -> None:
    announce(f"gated closed gates rows={rows} c={c} hidden={hidden} {dtype}")
    gen = torch.Generator(device=DEV).manual_seed(rows + c)
    normal = lambda scale, *shape: (torch.randn(shape, generator=gen, device=DEV) * scale).to(dtype)
    x, wg, wu, dh = normal(1.0, rows, c), normal(c ** -0.5, hidden, c), normal(c ** -0.5, hidden, c), normal(0.1, rows, hidden)
    x[:, 0], wg[:, 0], wu[:, 0] = 0.0, -1e10, 1e10
    far = [1, 3, rows - 1]
    x[far], dh[far] = 0.0, 1e19  # dh U leaves the range, too
    want = run(x, wg, wu, dh)
    for value in (1e10, 1e10 / 16):  # G = -1e20 and U = 1e20; 2^8 below
        x[far, 0] = value
        got = run(x, wg, wu, dh)
        assert not got[0][far].any() and not got[1][far].any()
        for name, a, b in zip(("h", "dx", "dgate", "dup"), got, want):
            assert torch.equal(a, b), name
