"""What the 16-bit gradients of the gated feed-forward product carry of rounding (``-m gpu``): dG and dU rounded to the type, as operands
of the products that follow, and the result rounded; nothing else of that size.

The same in 64 bits with these two roundings is the oracle.  A value that fp32 forms r of itself off falls to the other side of a
rounding border with the probability r / (2 E), and is then 2 E of itself off: 2-norm sqrt(2 E r), once for dG and dU and once
for the result.  Sums of up to 700 products are r = 4 sqrt(700) 2^-24 = 7e-6 off, so both together E / 10 (bf16, E = 2^-8) to E / 4 (fp16,
2^-11); E / 3 is asked.  A third rounding would be 0.4 E, and without the one of dG and dU the results would be 0.6 E off the oracle.
"""

from __future__ import annotations

import pytest
import torch
from test_gpu_gated_linear import announce, make

from omniwave_amd import gated_linear_hip

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,c,hidden", [(48, 512, 600), (700, 512, 256), (700, 128, 700), (300, 1536, 260)])
def test_two_roundings(rows, c, hidden, dtype) -> None:
    announce(f"gated roundings rows={rows} c={c} hidden={hidden} {dtype}")
    x, wg, wu, dh = make(rows, c, hidden, dtype)
    leaves = [t.requires_grad_(True) for t in (x, wg, wu)]
    got = torch.autograd.grad(gated_linear_hip(*leaves), leaves, dh)
    x, wg, wu, dh = (t.detach().double() for t in (x, wg, wu, dh))
    g, u = x @ wg.T, x @ wu.T
    s = torch.sigmoid(g)
    du, dg = ((v.to(dtype)).double() for v in (dh * g * s, dh * u * s * (1 + g * (1 - s))))
    e = torch.finfo(dtype).eps / 2
    for name, a, b in zip(("dx", "dgate", "dup"), got, (dg @ wg + du @ wu, dg.T @ x, du.T @ x)):
        off = (a.double() - b.to(dtype).double()).norm() / b.norm()
        assert off <= e / 3, f"{name}: {off.item()}"
