"""An infinity in a row of the norms (``-m gpu``), at every place of it, in rows whose channels fill whole vectors and
in others: by the formula the root of the mean is infinite, so what is finite in the row becomes zero under the
norm, the infinity itself NaN, and a weight's gradient has nothing of it but at its own channel.  Zeros, and
sums that an infinite row adds zeros to, are exact."""

from __future__ import annotations

import sys

import pytest
import torch

from omniwave_amd import block_norms_hip, rms_norm_hip

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
INF = float("inf")


def announce(msg: str) -> None:
    print(f"\n[gpu-case] {msg}", file=sys.stderr, flush=True)


def places(c: int) -> list[int]:
    return sorted({*range(min(c, 17)), *range(max(0, c - 17), c)})


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("c", [3, 5, 9, 13, 16, 95, 129, 1023, 2049, 4099, 8191, 8192])
def test_an_infinity_stays_where_it_is(c, dtype) -> None:
    announce(f"norms infinity c={c} {dtype}")
    dtype = TYPES[dtype]
    at = torch.tensor(places(c), device=DEV)
    rows = len(at)
    gen = torch.Generator(device=DEV).manual_seed(c)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=DEV).to(dtype)

    hit = at[:, None] == torch.arange(c, device=DEV)
    value = torch.where(torch.arange(rows, device=DEV) % 2 == 0, INF, -INF)[:, None]
    x, finite = normal(rows, c), normal(rows, c)
    bad = torch.where(hit, value, finite.float()).to(dtype)
    w = (torch.rand(c, generator=gen, device=DEV) + 0.5).to(dtype)

    weight = w.clone().requires_grad_(True)
    y = rms_norm_hip(bad, weight)
    assert y[hit].isnan().all() and not y[~hit].any()
    # Only these rows: every channel's sum is of zeros and, where the channel has an infinity, of NaN.
    (dw,) = torch.autograd.grad(y, weight, normal(rows, c))
    struck = hit.any(0)
    assert dw[struck].isnan().all() and not dw[~struck].any()

    post = w.clone().requires_grad_(True)
    out, nxt = block_norms_hip(x, bad, post_weight=post, next_weight=w)
    assert out[hit].isnan().all() and torch.equal(out[~hit], x[~hit])
    assert nxt.isnan().all()  # the row's mean square is NaN
    out, _ = block_norms_hip(x, bad, post_weight=post)
    (dpost,) = torch.autograd.grad(out, post, normal(rows, c))
    assert dpost[struck].isnan().all() and not dpost[~struck].any()
