"""Blocks and models with a norm after the block, on the CPU with the oracle as the backend, and the
training rows of the harness where there is no GPU."""

from __future__ import annotations

import pytest
import torch

from omniwave_amd import create_model
from omniwave_amd.block import OmniWeaveBlock, enable_fp8
from omniwave_amd.harness import run_benchmark
from oracle.bigemm import bigemm_delta_reference

SMALL = dict(widths=[32, 64, 128, 256], depths=[1, 1, 2, 1], channel_tiles=[32, 32, 64, 64], input_size=32)


def norm(x, w):
    return x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w


def make_block(**kw) -> OmniWeaveBlock:
    torch.manual_seed(0)
    block = OmniWeaveBlock(8, 8, 128, 64, "shifted", 0, backend="reference", post_norm=True, **kw)
    with torch.no_grad():
        block.gamma.uniform_(0.5, 1.5)
        block.norm_weight.uniform_(0.5, 1.5)
        block.post_norm_weight.uniform_(0.5, 1.5)
    return block


def test_block_is_the_formula(oracle_backend) -> None:
    block = make_block()
    x = torch.randn(2, 8, 8, 128)
    out = block(x)
    p = {k: v.detach().double() for k, v in block.named_parameters()}
    delta = bigemm_delta_reference(x=norm(x.double(), p["norm_weight"]), plan=block.plan,
                                   **{k: p[k] for k in ("a_u", "a_v", "a_o", "b_u", "b_v", "b_o")},
                                   gamma=torch.ones(128, dtype=torch.float64))
    want = x.double() + p["gamma"] * norm(delta, p["post_norm_weight"])
    # fp32 products of depth 16, 64, 128 and 16 and two norms: a few hundred half steps of 2^-24
    assert (out.double() - want).abs().max() <= 500 * 2 ** -24 * want.abs().max()


def test_gradients_of_the_branch(oracle_backend) -> None:
    """The norm's weight, LayerScale and the residual (the oracle backend itself has no gradient)."""
    block = make_block()
    x = torch.randn(2, 8, 8, 128, requires_grad=True)
    g = torch.randn(2, 8, 8, 128)
    block(x).backward(g)
    assert torch.equal(x.grad, g)
    with torch.no_grad():
        branch = (block(x) - x) / block.gamma
    assert torch.allclose(block.gamma.grad, (g * branch).sum((0, 1, 2)), rtol=1e-4, atol=1e-4)
    assert torch.allclose(block.post_norm_weight.grad, (g * block.gamma * branch / block.post_norm_weight).sum((0, 1, 2)),
                          rtol=1e-4, atol=1e-4)


def test_drop_path_scales_the_branch(oracle_backend) -> None:
    block = make_block(drop_path_rate=0.5).train()
    x = torch.randn(16, 8, 8, 128)
    torch.manual_seed(5)
    out = block(x) - x
    block.eval()
    whole = block(x) - x
    kept = [i for i in range(16) if out[i].abs().max() > 0]
    assert 0 < len(kept) < 16
    assert torch.allclose(out[kept], 2 * whole[kept], rtol=1e-5, atol=1e-5)


def test_the_default_model_has_no_such_parameters() -> None:
    plain, normed = create_model("omniweave_t", **SMALL), create_model("omniweave_t", post_norm=True, **SMALL)
    extra = set(normed.state_dict()) - set(plain.state_dict())
    assert extra == {f"stages.{i}.blocks.{j}.post_norm_weight" for i, n in enumerate(SMALL["depths"]) for j in range(n)}
    assert set(plain.state_dict()) < set(normed.state_dict())


def test_model_runs_and_trains(oracle_backend) -> None:
    model = create_model("omniweave_t", post_norm=True, num_classes=10, **SMALL)
    logits = model(torch.randn(2, 3, 32, 32))
    assert logits.shape == (2, 10)
    logits.sum().backward()
    assert model.stages[2].blocks[1].post_norm_weight.grad is not None
    with torch.no_grad():
        assert torch.equal(model(torch.ones(1, 3, 32, 32)), model(torch.ones(1, 3, 32, 32)))


def test_fp8_needs_the_hip_backend_and_eval(oracle_backend) -> None:
    block = make_block()
    enable_fp8(block, min_channel_tile=64)
    with pytest.raises(RuntimeError, match="inference-only"):
        block.train()(torch.randn(1, 8, 8, 128))
    with pytest.raises(RuntimeError, match="hip backend"):
        block.eval()(torch.randn(1, 8, 8, 128))


def test_training_rows_say_why_there_are_none() -> None:
    rows = run_benchmark({"resolutions": [32], "backends": [], "train_batch_sizes": [2], "warmup": 0, "iterations": 1},
                         torch.device("cpu"))
    assert [r["kind"] for r in rows] == ["train"]
    assert "error" in rows[0] and rows[0]["batch_size"] == 2


class Wrapped(torch.nn.Module):
    def __init__(self, inner) -> None:
        super().__init__()
        self.inner, self.calls = inner, 0

    def forward(self, x):
        self.calls += 1
        return self.inner(x)


@pytest.mark.parametrize("post_norm", [False, True])
def test_wrapped_blocks_and_hooks_are_called(oracle_backend, post_norm) -> None:
    model = create_model("omniweave_t", backend="reference", post_norm=post_norm, **SMALL)
    stage = model.stages[2]
    x = torch.randn(1, stage.blocks[0].plan.height, stage.blocks[0].plan.width, 128)
    want = stage(x)
    seen = []
    stage.blocks[0].register_forward_hook(lambda *_: seen.append(0))
    stage.blocks[1] = Wrapped(stage.blocks[1])
    assert torch.equal(stage(x), want) and seen == [0] and stage.blocks[1].calls == 1
