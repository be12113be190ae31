"""Layer norm, gated product and distillation together on the GPU (``-m gpu``), as a model and its training step call them.

Gates as the other model tests: rel-L2 1e-2 (bf16), 5e-3 (fp16) and 1e-4 (fp32) against the same in 64 bits on the same
weights, where a tensor is rounded to the type between the operators as here.
"""

from __future__ import annotations

import sys

import pytest
import torch

from omniwave_amd import create_model, cross_entropy_hip, distillation_hip
from omniwave_amd.feed_forward import GatedFeedForward
from omniwave_amd.harness import TrainingStep, run_benchmark

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
TOL = {torch.bfloat16: 1e-2, torch.float16: 5e-3, torch.float32: 1e-4}
MODEL = dict(widths=[64, 128, 128, 256], depths=[1, 2, 2, 1], channel_tiles=[64, 64, 128, 128], input_size=64,
             num_classes=100, layer_scale_init=0.5, feed_forward=1.5)


def announce(msg: str) -> None:
    print(f"\n[gpu-case] {msg}", file=sys.stderr, flush=True)


def rel(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm()).item()


class Rounded(torch.autograd.Function):
    """A tensor that is stored in the type, and whose gradient is."""

    @staticmethod
    def forward(ctx, x, dtype):
        ctx.dtype = dtype
        return x.to(dtype).double()

    @staticmethod
    def backward(ctx, g):
        return g.to(ctx.dtype).double(), None


def formula(p, x, dtype):
    r = lambda t: Rounded.apply(t, dtype)
    var, mean = torch.var_mean(x, -1, keepdim=True, correction=0)
    n = r((x - mean) / (var + 1e-6).sqrt() * p["norm_weight"] + p["norm_bias"])
    g = n @ p["gate.weight"].T
    h = r(g * torch.sigmoid(g) * (n @ p["up.weight"].T))
    return r(x + p["gamma"] * r(h @ p["down.weight"].T))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape,hidden", [((2, 7, 7, 256), 512), ((1, 1, 1, 64), 96), ((3, 10, 10, 95), 190), ((4, 28, 28, 128), 256)])
def test_block(shape, hidden, dtype) -> None:
    announce(f"feed-forward {shape} hidden={hidden} {dtype}")
    torch.manual_seed(0)
    block = GatedFeedForward(shape[-1], hidden, 0.5, "hip")
    with torch.no_grad():
        block.norm_weight.uniform_(0.5, 1.5)
        block.norm_bias.normal_(0, 0.1)
        block.gamma.uniform_(0.5, 1.5)
    block = block.to(device=DEV, dtype=dtype)
    x, up = (torch.randn(shape, device=DEV).to(dtype) for _ in range(2))
    x.requires_grad_(True)
    y = block(x)
    names, params = zip(*block.named_parameters())
    grads = torch.autograd.grad(y, (x, *params), up)
    p = {k: v.detach().double().requires_grad_(True) for k, v in zip(names, params)}
    xd = x.detach().double().requires_grad_(True)
    want = formula(p, xd, dtype)
    assert rel(y.detach(), want.detach()) <= TOL[dtype]
    for name, got, ref in zip(("x", *names), grads, torch.autograd.grad(want, (xd, *p.values()), up.double())):
        assert rel(got, ref) <= TOL[dtype], name


@pytest.mark.parametrize("x_dtype", [torch.bfloat16, torch.float32])
def test_block_under_autocast(x_dtype) -> None:
    """Weights of 32 bits: an x of 16 bits, as the layers before it return there, and one of 32."""
    announce(f"feed-forward under autocast x {x_dtype}")
    torch.manual_seed(0)
    block = GatedFeedForward(128, 200, 0.5, "hip").to(DEV)
    x, up = (torch.randn(3, 9, 9, 128, device=DEV).to(x_dtype) for _ in range(2))
    x.requires_grad_(True)
    with torch.autocast("cuda", torch.bfloat16):
        y = block(x)
    assert y.dtype == x_dtype
    names, params = zip(*block.named_parameters())
    grads = torch.autograd.grad(y, (x, *params), up)
    p = {k: v.detach().double().requires_grad_(True) for k, v in zip(names, params)}
    xd = x.detach().double().requires_grad_(True)
    want = formula(p, xd, torch.bfloat16)
    assert rel(y.detach(), want.detach()) <= TOL[torch.bfloat16]
    for name, got, ref in zip(("x", *names), grads, torch.autograd.grad(want, (xd, *p.values()), up.double())):
        assert got.dtype == (x_dtype if name == "x" else torch.float32) and rel(got, ref) <= TOL[torch.bfloat16], name


def make(dtype):
    torch.manual_seed(0)
    model = create_model("omniweave_t", backend="hip", **MODEL).to(device=DEV, dtype=dtype)
    images = torch.randn(6, 3, 64, 64, device=DEV).to(dtype)
    labels = torch.randint(0, 100, (6,), device=DEV)
    values, classes = (torch.randn(6, 100, device=DEV) * 3).topk(8, 1)
    classes[2, 5:], classes[4] = -100, -100  # a shorter list, an image without a teacher
    return model, images, labels, (values, classes)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_model_in_both_paths(dtype) -> None:
    announce(f"model with feed-forward {dtype}")
    model, images, _, _ = make(dtype)
    with torch.no_grad():
        fast = model(images)
    slow = model(images).detach()  # the path that keeps a graph
    assert rel(fast, slow) <= TOL[dtype]
    features = model.forward_features(images)
    stage = model.stages[0]
    with torch.no_grad():
        before = stage._forward_plain(model._stem(images))
        p = {k: v.detach().double() for k, v in stage.feed_forward.named_parameters()}
        assert rel(features["stage1"].detach(), formula(p, before.double(), dtype)) <= TOL[dtype]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_training_step_with_a_teacher(dtype) -> None:
    """The step's loss and gradients are those of its parts; every parameter moves."""
    announce(f"training step with a teacher {dtype}")
    model, images, labels, teacher = make(dtype)
    training = TrainingStep(model, distill_weight=0.3, temperature=2.0, max_grad_norm=None, master_weights=dtype != torch.float32)
    logits = model(images)
    leaf = logits.detach().requires_grad_(True)
    parts = [cross_entropy_hip(leaf, labels, label_smoothing=0.1), distillation_hip(leaf, *teacher, temperature=2.0)]
    want = 0.7 * parts[0] + 0.3 * parts[1]
    up = torch.autograd.grad(want, leaf)[0]
    params = dict(model.named_parameters())
    grads = dict(zip(params, torch.autograd.grad(logits, list(params.values()), up)))
    before = {k: v.detach().clone() for k, v in params.items()}
    loss = training.step(images, labels, teacher=teacher)
    assert abs(loss.item() - want.item()) <= 1e-5 * abs(want.item())
    for name, p in params.items():
        assert p.grad.isfinite().all(), name
        # the logits' gradient is a sum of two rounded ones there
        assert rel(p.grad, grads[name]) <= 3 * TOL[dtype], name
    # AdamW's first step moves every value with a gradient by the learning rate, 1e-3
    for name, p in params.items():
        if dtype == torch.float32:
            assert (p.detach() - before[name]).abs().max().item() > 1e-4, name
    # a weight of 0 is the labels' loss alone
    training.distill_weight = 0.0
    with torch.no_grad():
        alone = cross_entropy_hip(model(images), labels, label_smoothing=0.1)
    assert abs(training.step(images, labels, teacher=teacher).item() - alone.item()) <= 2 * TOL[dtype] * alone.item()


def test_training_rows() -> None:
    announce("training rows with feed-forward and a teacher")
    options = {k: v for k, v in MODEL.items() if k not in ("input_size", "num_classes")}
    rows = run_benchmark({"resolutions": [64], "train_batch_sizes": [4], "latency_batch_sizes": [], "throughput_batch_sizes": [],
                          "warmup": 1, "iterations": 2, "train_teacher_top": 5, "model_options": options}, DEV)
    assert len(rows) == 1 and "error" not in rows[0], rows
    assert rows[0]["images_per_second"] > 0


def test_a_captured_step_of_all_three() -> None:
    """Norm, gated product, projection, residual and loss with their backward in one graph, replayed with other inputs."""
    announce("captured feed-forward and distillation")
    torch.manual_seed(0)
    block = GatedFeedForward(64, 128, 0.5, "hip").to(device=DEV, dtype=torch.bfloat16)
    head = torch.randn(50, 64, device=DEV).bfloat16()
    x = torch.randn(3, 25, 64, device=DEV).bfloat16().requires_grad_(True)
    values, classes = torch.randn(75, 50, device=DEV).topk(6, 1)
    params = [x, *block.parameters()]

    def step():
        loss = distillation_hip(block(x).reshape(75, 64) @ head.T, values, classes, temperature=2.0)
        return loss.detach(), *torch.autograd.grad(loss, params)

    step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for n in range(3):
        with torch.no_grad():
            x.mul_(0.9)
            classes.copy_(classes.roll(1, 0))
            block.norm_bias.add_(0.1)
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        torch.cuda.synchronize()
        for a, b in zip(held, eager):
            assert torch.equal(a, b), f"replay {n}"
