"""``AdamW.grad_norm`` is the last step's, also of a step that finds no gradient or clips nothing (on the CPU)."""

from __future__ import annotations

import torch

from omniwave_amd import AdamW


def test_no_gradients_have_a_norm_of_zero() -> None:
    p, empty = torch.nn.Parameter(torch.ones(3)), torch.nn.Parameter(torch.ones(0))
    opt = AdamW([p, empty], max_grad_norm=1.0)
    for empty.grad in (None, torch.ones(0)):
        opt.grad_norm = torch.tensor(5.0)  # of the step before
        opt.step()
        assert opt.grad_norm.shape == () and opt.grad_norm.dtype == torch.float32 and opt.grad_norm.item() == 0.0
    assert torch.equal(p.detach(), torch.ones(3))


def test_no_parameters_at_all() -> None:
    opt = AdamW([{"params": []}], max_grad_norm=1.0)
    opt.step()
    assert opt.grad_norm.item() == 0.0


def test_no_clip_has_no_norm() -> None:
    opt = AdamW([torch.nn.Parameter(torch.ones(3))], max_grad_norm=1.0)
    opt.step()
    opt.max_grad_norm, opt.grad_norm = None, torch.tensor(5.0)
    opt.step()
    assert opt.grad_norm is None
