"""A training step of the framework's operators together on the GPU (``-m gpu``): blocks and models with a
norm after the block, the cross-entropy, the backward and the AdamW step.

Gates as the other model tests: rel-L2 1e-2 (bf16), 5e-3 (fp16) and 1e-4 (fp32) against an fp32 composition of
the same step, whose BiGEMM is the oracle's on the CPU.
"""

from __future__ import annotations

import copy
import sys

import pytest
import torch
import torch.nn.functional as F

from omniwave_amd import AdamW, create_model, cross_entropy_hip
from omniwave_amd.block import OmniWeaveBlock, enable_fp8
from omniwave_amd.harness import TrainingStep, run_benchmark
from omniwave_amd.hip import bigemm_block_hip
from oracle.bigemm import bigemm_delta_reference, rel_l2

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
TOL = {torch.bfloat16: 1e-2, torch.float16: 5e-3, torch.float32: 1e-4}
MODEL = dict(widths=[64, 128, 128, 256], depths=[1, 2, 2, 1], channel_tiles=[64, 64, 128, 128], input_size=64,
             num_classes=100, layer_scale_init=0.5, post_norm=True)


def announce(msg: str) -> None:
    print(f"\n[gpu-case] {msg}", file=sys.stderr, flush=True)


def norm(x, w):
    return x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w


def make_block(h, c, d, route, level, dtype, **kw) -> OmniWeaveBlock:
    torch.manual_seed(0)
    block = OmniWeaveBlock(h, h, c, d, route, level, backend="hip", post_norm=True, **kw)
    with torch.no_grad():
        for p in (block.gamma, block.norm_weight, block.post_norm_weight):
            p.uniform_(0.5, 1.5)
        block.b_u.normal_(0.0, d ** -0.5)
        block.b_v.normal_(0.0, d ** -0.5)
        block.b_o.normal_(0.0, (2 * d) ** -0.5)
    return block.to(device=DEV, dtype=dtype)


def reference(block, x, scale=None, noise=0.0):
    """The block in fp32 on the CPU, its delta and delta's gradient off by up to ``noise`` of themselves;
    returns its output and the leaves."""
    p = {k: v.detach().float().cpu().requires_grad_(True) for k, v in block.named_parameters()}
    x = x.detach().float().cpu().requires_grad_(True)
    delta = bigemm_delta_reference(x=norm(x, p["norm_weight"]), plan=block.plan,
                                   **{k: p[k] for k in ("a_u", "a_v", "a_o", "b_u", "b_v", "b_o")}, gamma=torch.ones(x.shape[-1]))
    if noise:
        off = [1 + noise * (2 * torch.rand(delta.shape, generator=torch.Generator().manual_seed(n)) - 1) for n in (9, 10)]
        delta.register_hook(lambda grad: grad * off[1])
        delta = delta * off[0]
    branch = p["gamma"] * norm(delta, p["post_norm_weight"])
    if scale is not None:
        branch = branch * scale.cpu().reshape(-1, 1, 1, 1)
    return x + branch, {"x": x, **p}


@pytest.mark.parametrize("h,c,d,route,level,dtype", [
    (28, 256, 64, "local", 0, torch.bfloat16), (14, 512, 128, "shifted", 0, torch.bfloat16),
    (14, 256, 128, "radix", 1, torch.float16), (7, 96, 64, "local", 0, torch.bfloat16), (14, 256, 64, "shifted", 0, torch.float32),
])
def test_block_forward_and_backward(h, c, d, route, level, dtype) -> None:
    announce(f"post-norm block {h}x{h}x{c} {route}{level} {dtype}")
    block = make_block(h, c, d, route, level, dtype)
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(2, h, h, c, generator=gen).to(dtype).to(DEV).requires_grad_(True)
    g = torch.randn(2, h, h, c, generator=gen).to(dtype).to(DEV)
    out = block(x)
    out.backward(g)
    want, leaves = reference(block, x)
    want.backward(g.float().cpu())
    assert rel_l2(out.detach().cpu().float() - x.detach().cpu().float(), (want - leaves["x"]).detach()) <= TOL[dtype]
    assert rel_l2(x.grad.cpu().float() - g.cpu().float(), leaves["x"].grad - g.cpu().float()) <= TOL[dtype]
    # The norm divides a row by its own size: a row whose delta is small (at 7x7 the 49th token is alone in its
    # group, and its delta is a product of two single token weights, 200 times below the others') hands
    # the BiGEMM's rounding on that much larger, and its exact derivative by those weights' scale is zero, so
    # what it adds to their gradient is rounding alone.  The BiGEMM's gate therefore comes on top as what a delta
    # and a gradient of it within that gate do to the oracle's own gradient.
    moved, other = reference(block, x, noise=TOL[dtype])
    moved.backward(g.float().cpu())
    for name, p in block.named_parameters():
        allowed = TOL[dtype] + rel_l2(other[name].grad, leaves[name].grad)
        assert allowed <= 10 * TOL[dtype] and rel_l2(p.grad.cpu().float(), leaves[name].grad) <= allowed, name


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_block_gradients_equal_the_composition(dtype) -> None:
    """The same BiGEMM with the norm, LayerScale and residual in fp32 torch operations: apart by the rounding of
    dx and delta's gradient to the activation dtype, and fp32's."""
    announce(f"post-norm block against composition {dtype}")
    block = make_block(7, 96, 64, "local", 0, dtype)
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(2, 7, 7, 96, generator=gen).to(dtype).to(DEV).requires_grad_(True)
    g = torch.randn(2, 7, 7, 96, generator=gen).to(dtype).to(DEV)
    block(x).backward(g)
    ours = {n: p.grad.clone() for n, p in block.named_parameters()}
    block.zero_grad()
    b = block
    delta = bigemm_block_hip(x, b.norm_weight, b.plan, b.a_u, b.a_v, b.a_o, b.b_u, b.b_v, b.b_o, b._ones, residual=False)
    (x.float() + b.gamma.float() * norm(delta.float(), b.post_norm_weight.float())).backward(g.float())
    gate = 2 * torch.finfo(dtype).eps + 1e-5
    for n, p in block.named_parameters():
        assert rel_l2(ours[n].float().cpu(), p.grad.float().cpu()) <= gate, n


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_row_of_blocks_equals_the_blocks(dtype) -> None:
    """A stage hands each block its normalised input from the block before it; block by block the norm is the
    BiGEMM kernel's, which rounds its statistics to the activation dtype."""
    announce(f"post-norm stage {dtype}")
    torch.manual_seed(0)
    model = create_model("omniweave_t", backend="hip", **MODEL).to(device=DEV, dtype=dtype)
    stage = model.stages[2]
    x = torch.randn(4, 4, 4, 128, device=DEV).to(dtype)
    calls = []
    whole = stage._forward_normed
    stage._forward_normed = lambda t: calls.append(1) or whole(t)
    with torch.no_grad():
        row = stage(x)
        y = stage.anchor(x)
        for block in stage.blocks:
            y = block(y)
    assert calls
    assert rel_l2((row - x).float().cpu(), (y - x).float().cpu()) <= TOL[dtype]


def test_drop_path_of_a_row_of_blocks() -> None:
    announce("post-norm drop-path")
    block = make_block(14, 256, 128, "local", 0, torch.float32, drop_path_rate=0.4).train()
    x = torch.randn(8, 14, 14, 256, device=DEV)
    torch.manual_seed(3)
    out = block(x)
    torch.manual_seed(3)
    scale = torch.empty((8, 1, 1, 1), device=DEV).bernoulli_(0.6).reshape(8) / 0.6
    want, leaves = reference(block, x, scale)
    assert 0 < (scale > 0).sum() < 8
    assert torch.equal(out[scale == 0], x[scale == 0])
    assert rel_l2((out - x).detach().cpu(), (want - leaves["x"]).detach()) <= 1e-4


def test_fp8_blocks_keep_their_norm_fused() -> None:
    announce("post-norm fp8")
    block = make_block(14, 512, 128, "local", 0, torch.bfloat16).eval()
    x = torch.randn(2, 14, 14, 512, device=DEV).bfloat16()
    with torch.no_grad():
        plain = block(x)
        enable_fp8(block)
        assert not block.takes_normed(x)
        fp8 = block(x)
    err = rel_l2((fp8 - x).float().cpu(), (plain - x).float().cpu())
    assert 0 < err <= 8e-2


class Composed(torch.nn.Module):
    """The model with its BiGEMMs, and everything else as torch operations in fp32."""

    def __init__(self, model) -> None:
        super().__init__()
        self.model = model

    def forward(self, images):
        m = self.model
        x = m._stem(images)
        for i, stage in enumerate(m.stages):
            if stage.anchor is not None:
                x = stage.anchor(x)
            for b in stage.blocks:
                delta = bigemm_block_hip(x, b.norm_weight, b.plan, b.a_u, b.a_v, b.a_o, b.b_u, b.b_v, b.b_o, b._ones,
                                         residual=False)
                x = x + b.gamma * norm(delta, b.post_norm_weight)
            if i < 3:
                n, h, w, c = x.shape
                x = x.reshape(n, h // 2, 2, w // 2, 2, c).permute(0, 1, 3, 2, 4, 5).reshape(n, h // 2, w // 2, 4 * c)
                x = m.downsamples[i](x)
        return m.head(x.mean(dim=(1, 2)))


def test_step_of_a_model_against_torch() -> None:
    """Loss and every gradient of a mixed-label step in fp32, then the AdamW step of those gradients beside
    torch's (both round in fp32 alone: 24 half steps of an update of at most lr, 3 of the parameter)."""
    announce("training step against torch")
    torch.manual_seed(0)
    ours = create_model("omniweave_t", backend="hip", **MODEL).to(DEV)
    theirs = copy.deepcopy(ours)
    gen = torch.Generator().manual_seed(1)
    images = torch.randn(4, 3, 64, 64, generator=gen).to(DEV)
    a, b = (torch.randint(0, 100, (4,), generator=gen).to(DEV) for _ in range(2))
    loss = cross_entropy_hip(ours(images), a, target_b=b, mix=0.7, label_smoothing=0.1)
    loss.backward()
    logits = Composed(theirs)(images)
    want = 0.7 * F.cross_entropy(logits, a, label_smoothing=0.1) + 0.3 * F.cross_entropy(logits, b, label_smoothing=0.1)
    want.backward()
    assert abs(loss.item() - want.item()) <= 1e-5 * want.item()
    for (name, p), q in zip(ours.named_parameters(), theirs.parameters()):
        assert rel_l2(p.grad.cpu(), q.grad.cpu()) <= 1e-4, name
        q.grad.copy_(p.grad)
    first, second = AdamW(ours.parameters(), lr=1e-3), torch.optim.AdamW(theirs.parameters(), lr=1e-3, foreach=False)
    first.step(), second.step()
    u = 2.0 ** -24
    for (name, p), q in zip(ours.named_parameters(), theirs.parameters()):
        bound = 2 * (24 * u * 1e-3 + 3 * u * p.detach().abs())
        assert ((p - q).detach().abs() <= bound).all(), name


def test_the_next_forward_sees_the_step() -> None:
    """The BiGEMM packs its weights once per version of the parameters."""
    announce("step seen by packed weights")
    block = make_block(14, 256, 128, "local", 0, torch.bfloat16)
    x = torch.randn(2, 14, 14, 256, device=DEV).bfloat16()
    opt = AdamW(block.parameters(), lr=0.05)
    for _ in range(2):
        block(x).float().square().mean().backward()
        versions = [p._version for p in block.parameters()]
        opt.step()
        assert all(p._version > v for p, v in zip(block.parameters(), versions))
        with torch.no_grad():
            got = block(x)
            fresh = copy.deepcopy(block)(x)
        assert torch.equal(got, fresh)


@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, 8), (torch.bfloat16, 32), (torch.float32, 32)])
def test_training_steps_run_and_repeat(dtype, bits) -> None:
    announce(f"training steps {dtype} bits={bits}")
    gen = torch.Generator().manual_seed(2)
    images = torch.randn(8, 3, 64, 64, generator=gen).to(DEV).to(dtype)
    labels = torch.randint(0, 100, (8,), generator=gen).to(DEV)
    runs = []
    for _ in range(2):
        torch.manual_seed(0)
        model = create_model("omniweave_t", backend="hip", **MODEL).to(device=DEV, dtype=dtype).train()
        training = TrainingStep(model, state_bits=bits)
        losses = [training.step(images, labels) for _ in range(4)]
        assert all(torch.isfinite(v) for v in losses)
        moved = [p.detach().clone() for p in model.parameters()]
        assert all(torch.isfinite(p).all() for p in moved)
        runs.append([*losses, *moved])
    assert sum(torch.equal(a, b) for a, b in zip(*runs)) == len(runs[0])


def test_training_rows() -> None:
    announce("harness training rows")
    options = {k: v for k, v in MODEL.items() if k != "input_size"}
    rows = run_benchmark({"resolutions": [64], "backends": [], "train_batch_sizes": [4], "train_dtypes": ["bfloat16", "float32"],
                          "model_options": options, "training": {"state_bits": 8}, "warmup": 1, "iterations": 2}, DEV)
    assert len(rows) == 2 and all("error" not in r for r in rows), rows
    assert all(r["kind"] == "train" and r["images_per_second"] > 0 for r in rows)


def test_hooks_and_wrappers_of_blocks_are_called() -> None:
    """The stage runs its blocks one by one where something listens; the two ways differ by roundings of the
    normalised inputs (half a step of bf16 each, through two blocks)."""
    announce("post-norm stage with hooks")
    torch.manual_seed(0)
    model = create_model("omniweave_t", backend="hip", post_norm=True).to(DEV, torch.bfloat16).train()
    stage = model.stages[2]
    x = torch.randn(2, 14, 14, stage.blocks[0].dim, device=DEV).bfloat16()
    assert stage._takes_normed(x)
    want = stage(x)
    seen = []
    handle = stage.blocks[1].register_forward_hook(lambda *_: seen.append(1))
    assert not stage._takes_normed(x)
    got = stage(x)
    assert seen == [1]
    assert (got.float() - want.float()).norm() <= 2e-2 * want.float().norm()
    handle.remove()
    assert stage._takes_normed(x) and torch.equal(stage(x), want)
    inner = stage.blocks[0]
    stage.blocks[0] = torch.nn.Sequential(inner)
    assert not stage._takes_normed(x) and torch.equal(stage(x), got)
