"""The package imports and its shortcuts step aside where torch has not the internal names by which they see that nobody
listens to a call (on the CPU, in a process of its own)."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent

BLOCK = """
import torch.nn.modules.module as m
del m._has_any_global_hook
import torch, omniwave_amd
from omniwave_amd.block import OmniWeaveBlock
block = OmniWeaveBlock(height=8, width=8, dim=128, channel_tile=64, route="local", radix_level=0, post_norm=True)
block._fused = lambda x: True
assert not block.takes_normed(torch.zeros(1, 8, 8, 128))  # the block is called like any module
"""

# The name is missing while the package is imported; torch's own functions then go on using theirs.
OPTIMIZER = """
import torch
from torch.optim import optimizer as base
owner, name = {owner}, "{name}"
kept = vars(owner)[name]
delattr(owner, name)
import omniwave_amd
setattr(owner, name, kept)
p = torch.nn.Parameter(torch.ones(3))
opt = omniwave_amd.AdamW([p])
heard = []
opt.register_step_pre_hook(lambda *a: heard.append("before"))
opt.register_step_post_hook(lambda *a: heard.append("after"))
opt.step()
assert heard == ["before", "after"], heard
assert opt.step(lambda: 5) == 5
torch.optim.lr_scheduler.StepLR(opt, 1).step()
"""


def run(text: str) -> None:
    done = subprocess.run([sys.executable, "-c", text], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_global_hooks_of_modules() -> None:
    run(BLOCK)


@pytest.mark.parametrize("owner,name", [
    ("base", "_global_optimizer_pre_hooks"), ("base", "_global_optimizer_post_hooks"),
    ("torch.optim.Optimizer", "profile_hook_step"), ("torch.autograd.profiler", "_is_profiler_enabled")])
def test_hooks_of_optimizers(owner, name) -> None:
    run(OPTIMIZER.format(owner=owner, name=name))
