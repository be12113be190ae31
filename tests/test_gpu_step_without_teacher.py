"""A training step whose batch has no teacher's entry, or whose weight for the teacher is 0 (``-m gpu``)."""

from __future__ import annotations

import sys

import pytest
import torch

from omniwave_amd import create_model, cross_entropy_hip, distillation_hip
from omniwave_amd.harness import TrainingStep

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
MODEL = dict(widths=[64, 128, 128, 256], depths=[1, 1, 1, 1], channel_tiles=[64, 64, 128, 128], input_size=64,
             num_classes=100)


def announce(msg: str) -> None:
    print(f"\n[gpu-case] {msg}", file=sys.stderr, flush=True)


def make():
    torch.manual_seed(0)
    model = create_model("omniweave_t", backend="hip", feed_forward=1.0, **MODEL).to(DEV)
    images = torch.randn(4, 3, 64, 64, device=DEV)
    labels = torch.randint(0, 100, (4,), device=DEV)
    values, classes = (torch.randn(4, 100, device=DEV) * 3).topk(6, 1)
    return model, images, labels, values, classes


def reference(model, images, labels):
    with torch.no_grad():
        return cross_entropy_hip(model(images), labels, label_smoothing=0.1).item()


def none_by_class(v, i):
    return v, torch.full_like(i, -100)


def none_by_logit(v, i):
    return torch.full_like(v, -float("inf")), i


def of_no_entries(v, i):
    return v[:, :0], i[:, :0]


@pytest.mark.parametrize("without", [none_by_class, none_by_logit, of_no_entries])
def test_a_batch_without_a_teacher(without) -> None:
    """The labels' part of the loss stays, and the gradients are those of it.  Both losses come from models whose paths differ
    (with and without a graph), in fp32: 1e-4 of them."""
    announce(f"step of a batch without a teacher: {without.__name__}")
    model, images, labels, v, i = make()
    want = reference(model, images, labels)
    training = TrainingStep(model, distill_weight=0.25, max_grad_norm=None)
    loss = training.step(images, labels, teacher=without(v, i))
    assert abs(loss.item() - 0.75 * want) <= 1e-4 * want
    grads = {k: p.grad.clone() for k, p in model.named_parameters()}
    model, images, labels, *_ = make()  # the same anew
    logits = model(images)
    (0.75 * cross_entropy_hip(logits, labels, label_smoothing=0.1)).backward()
    for name, p in model.named_parameters():
        assert grads[name].isfinite().all()
        assert (grads[name] - p.grad).norm() <= 1e-5 * p.grad.norm() + 1e-12, name


def test_no_weight_for_the_teacher() -> None:
    """The loss is the labels', whatever the teacher says."""
    announce("step with no weight for the teacher")
    model, images, labels, v, i = make()
    v[1, 2] = float("nan")
    for teacher in ((v, i), none_by_class(v, i)):
        want = reference(model, images, labels)
        loss = TrainingStep(model, distill_weight=0.0, max_grad_norm=None).step(images, labels, teacher=teacher)
        assert abs(loss.item() - want) <= 1e-4 * want
        assert all(p.grad.isfinite().all() for p in model.parameters())


def test_a_teacher_that_is_no_number_shows() -> None:
    announce("step with a teacher that is no number")
    for bad in (dict(v=float("nan")), dict(i=100)):
        model, images, labels, v, i = make()
        i[1:] = -100
        if "v" in bad:
            v[0, 3] = bad["v"]
        else:
            i[0, 3] = bad["i"]
        assert TrainingStep(model, max_grad_norm=None).step(images, labels, teacher=(v, i)).isnan()


def test_no_weight_for_the_labels() -> None:
    """Labels that are all left out make no NaN of the teacher's loss."""
    announce("loss with no weight for the labels")
    model, images, labels, v, i = make()
    logits = model(images).detach().requires_grad_(True)
    loss = TrainingStep(model, distill_weight=1.0).loss(logits, torch.full_like(labels, -100), teacher=(v, i))
    (grad,) = torch.autograd.grad(loss, logits)
    assert torch.equal(loss.detach(), distillation_hip(logits.detach(), v, i)) and grad.isfinite().all() and grad.any()


def test_a_teacher_that_is_refused() -> None:
    announce("step with a teacher of other classes")
    model, images, labels, v, i = make()
    with pytest.raises(ValueError, match="teacher_indices"):
        TrainingStep(model).step(images, labels, teacher=(v, i.int()))


def test_captured() -> None:
    """The loss and its gradient, captured: replays of batches with and without entries in turn."""
    announce("captured loss of batches without a teacher")
    model, _, labels, v, i = make()
    training = TrainingStep(model, temperature=2.0)
    logits = torch.randn(4, 100, device=DEV, requires_grad=True)

    def run():
        loss = training.loss(logits, labels, teacher=(v, i))
        return loss.detach(), torch.autograd.grad(loss, logits)[0]

    run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    full, none = i.clone(), torch.full_like(i, -100)
    for n in range(4):
        i.copy_(full if n % 2 else none)
        graph.replay()
        torch.cuda.synchronize()
        eager = run()
        torch.cuda.synchronize()
        assert all(a.isfinite().all() and torch.equal(a, b) for a, b in zip(held, eager)), f"replay {n}"
