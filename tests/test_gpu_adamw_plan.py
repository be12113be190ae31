"""A step of AdamW (``-m gpu``) whose parameter is another view of its memory than in the step before is refused
before anything is launched: nothing in that memory and no state changes."""

from __future__ import annotations

import sys

import pytest
import torch

from omniwave_amd import AdamW

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def announce(msg: str) -> None:
    print(f"\n[gpu-case] {msg}", file=sys.stderr, flush=True)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("how", ["narrowed", "transposed", "retyped"])
def test_changed_views_are_refused(how, bits) -> None:
    announce(f"adamw changed view {how} bits={bits}")
    p, q = (torch.nn.Parameter(torch.randn(80, 80, device=DEV)) for _ in range(2))
    opt = AdamW([q, p], lr=0.1, state_bits=bits, max_grad_norm=1.0)
    for t in (p, q):
        t.grad = torch.randn_like(t)
    opt.step()
    whole = p.data
    p.grad = None
    p.data = {"narrowed": whole[:7], "transposed": whole.t(), "retyped": whole.view(torch.bfloat16)}[how]
    p.grad = torch.ones(p.shape, dtype=p.dtype, device=DEV)
    assert p.data_ptr() == whole.data_ptr()
    kept = [whole.clone(), q.detach().clone(), *[v.clone() for t in (p, q) for v in opt.state[t].values()]]
    with pytest.raises(ValueError):
        opt.step()
    found = [whole, q.detach(), *[v for t in (p, q) for v in opt.state[t].values()]]
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(found, kept))
    p.grad = None  # as it was, the step goes on
    p.data = whole
    p.grad = torch.ones_like(p)
    opt.step()
    assert not torch.equal(whole, kept[0]) and (opt.state[p]["step"] == 2).all()
