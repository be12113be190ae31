"""Gated feed-forward product on the GPU (``-m gpu``) in every kernel of its products (``test_gated_plans.py`` says which a size
takes), against the formula in 64 bits with the bounds of ``test_gpu_gated_linear.py``, and twice with the same bits."""

from __future__ import annotations

import pytest
import torch
from test_gated_plans import CASES, plans
from test_gpu_gated_linear import TYPES, announce, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,c,hidden,narrow,wide", CASES)
def test_every_kernel(rows, c, hidden, narrow, wide, dtype) -> None:
    announce(f"gated plans rows={rows} c={c} hidden={hidden} {dtype}")
    assert ", ".join(plans(rows, c, hidden, dtype)) == (wide if dtype == "f32" else narrow)
    given = make(rows, c, hidden, TYPES[dtype])
    first = check(*given)
    assert all(torch.equal(a, b) for a, b in zip(first, check(*given)))
