"""The operators of a training step past 32-bit offsets and in unusual calls (``-m gpu``)."""

from __future__ import annotations

import sys

import pytest
import torch

from omniwave_amd import AdamW, block_norms_hip, cross_entropy_hip, rms_norm_hip

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def announce(msg: str) -> None:
    print(f"\n[gpu-case] {msg}", file=sys.stderr, flush=True)


def test_norms_past_32_bit_offsets() -> None:
    """2.25e9 values: 550 copies of the same rows give 550 copies of their results, to the bit."""
    announce("norms of 2.25e9 values")
    gen = torch.Generator(device=DEV).manual_seed(0)
    small = [torch.randn(1, 4000, 1024, generator=gen, device=DEV).bfloat16().requires_grad_(True) for _ in range(2)]
    up = [torch.randn(1, 4000, 1024, generator=gen, device=DEV).bfloat16() for _ in range(2)]
    w = [torch.rand(1024, generator=gen, device=DEV) + 0.5 for _ in range(3)]
    call = lambda x, d: block_norms_hip(x, d, post_weight=w[0], gate=w[1], next_weight=w[2])
    outs = call(*small)
    want = [*[o.detach() for o in outs], *torch.autograd.grad(outs, small, up)]
    large = [t.detach().expand(550, 4000, 1024).contiguous().requires_grad_(True) for t in small]
    assert large[0].numel() > 1 << 31
    outs = call(*large)
    # upstream rows repeat: an expanded tensor of another image stride than row stride, copied by the call
    grads = torch.autograd.grad(outs, large, [g.expand(550, 4000, 1024) for g in up])
    for got, ref in zip((*[o.detach() for o in outs], *grads), want):
        for image in (0, 261, 262, 523, 524, 549):  # around 2^30 and 2^31 values, the last
            assert torch.equal(got[image], ref[0])


def test_cross_entropy_past_32_bit_offsets() -> None:
    announce("cross-entropy of 2.3e9 logits")
    gen = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(1000, 33001, generator=gen, device=DEV).bfloat16()
    a = torch.randint(0, 33001, (1000,), generator=gen, device=DEV)
    small = x.clone().requires_grad_(True)
    losses = cross_entropy_hip(small, a, reduction="sum", label_smoothing=0.1)
    (want,) = torch.autograd.grad(losses, small)
    large = x.repeat(70, 1).requires_grad_(True)
    assert large.numel() > 1 << 31
    labels = a.repeat(70)
    labels[:-1000] = -100  # the last rows alone count
    loss = cross_entropy_hip(large, labels, reduction="sum", label_smoothing=0.1)
    (grad,) = torch.autograd.grad(loss, large)
    assert torch.equal(grad[-1000:], want) and not grad[:1000].any()
    assert abs(loss.item() - losses.item()) <= 1e-6 * losses.item()


def test_adamw_past_32_bit_offsets() -> None:
    announce("adamw of 2.15e9 values")
    n = (1 << 31) + 3 * 4096 + 77
    tail = 2 * 4096 + 77  # begins at a chunk
    gen = torch.Generator(device=DEV).manual_seed(0)
    p = torch.nn.Parameter(torch.zeros(n, dtype=torch.bfloat16, device=DEV))
    p.grad = torch.zeros_like(p)
    q = torch.nn.Parameter(torch.randn(tail, generator=gen, device=DEV).bfloat16())
    opt, ref = AdamW([p], state_bits=8), AdamW([q], state_bits=8)
    with torch.no_grad():
        p[-tail:].copy_(q)
    for _ in range(3):
        q.grad = torch.randn(tail, generator=gen, device=DEV).bfloat16()
        p.grad[-tail:].copy_(q.grad)
        opt.step(), ref.step()
        assert torch.equal(p[-tail:], q)
    a, b = opt.state[p], ref.state[q]
    assert torch.equal(a["exp_avg"][-tail:].float(), b["exp_avg"].float())
    assert torch.equal(a["exp_avg_sq_root_scale"][-b["exp_avg_sq_root_scale"].numel():], b["exp_avg_sq_root_scale"])
    assert not p[:-tail].any() and (a["step"] == 3).all()


def test_the_same_tensor_in_two_places() -> None:
    announce("norms of x and x, one weight twice")
    gen = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(2, 9, 96, generator=gen, device=DEV, requires_grad=True)
    w = (torch.rand(96, generator=gen, device=DEV) + 0.5).requires_grad_(True)
    g = torch.randn(2, 9, 96, generator=gen, device=DEV)
    out, nxt = block_norms_hip(x, x, post_weight=w, gate=w, next_weight=w)
    both = torch.autograd.grad((out, nxt), (x, w), (g, g))
    parts = [x.detach().clone().requires_grad_(True) for _ in range(2)], [w.detach().clone().requires_grad_(True) for _ in range(3)]
    outs = block_norms_hip(*parts[0], post_weight=parts[1][0], gate=parts[1][1], next_weight=parts[1][2])
    grads = torch.autograd.grad(outs, (*parts[0], *parts[1]), (g, g))
    assert torch.equal(out, outs[0]) and torch.equal(nxt, outs[1])
    assert torch.allclose(both[0], grads[0] + grads[1], rtol=1e-6, atol=1e-6)
    assert torch.allclose(both[1], grads[2] + grads[3] + grads[4], rtol=1e-5, atol=1e-5)


def test_orders_and_broadcasts_that_are_copied() -> None:
    announce("norms of transposed rows, expanded gates")
    gen = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(3, 96, 7, generator=gen, device=DEV, requires_grad=True)
    d = torch.randn(3, 96, 7, generator=gen, device=DEV, requires_grad=True)
    gate = torch.rand(1, 96, generator=gen, device=DEV, requires_grad=True)
    w = torch.rand(192, generator=gen, device=DEV, requires_grad=True)
    g = torch.randn(3, 7, 96, generator=gen, device=DEV)

    def call(x, d, gate, w):
        return block_norms_hip(x, d, post_weight=w, gate=gate, next_weight=w)

    got = call(x.transpose(1, 2), d.transpose(1, 2), gate.expand(3, 96), w[::2])
    grads = torch.autograd.grad(got, (x, d, gate, w), (g, g))
    flat = [t.detach().transpose(1, 2).contiguous().requires_grad_(True) for t in (x, d)]
    gate3, half = gate.detach().expand(3, 96).contiguous().requires_grad_(True), w.detach()[::2].contiguous().requires_grad_(True)
    want = call(*flat, gate3, half)
    ref = torch.autograd.grad(want, (*flat, gate3, half), (g, g))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(grads[0], ref[0].transpose(1, 2)) and torch.equal(grads[1], ref[1].transpose(1, 2))
    assert torch.allclose(grads[2], ref[2].sum(0, keepdim=True), rtol=1e-5, atol=1e-5)
    assert torch.equal(grads[3][::2], ref[3]) and not grads[3][1::2].any()


def test_half_precision_mix_and_numbers_of_other_kinds() -> None:
    announce("cross-entropy argument kinds")
    gen = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(6, 50, generator=gen, device=DEV)
    a, b = (torch.randint(0, 50, (6,), generator=gen, device=DEV) for _ in range(2))
    mix = torch.rand(6, generator=gen, device=DEV).bfloat16()
    one = cross_entropy_hip(x, a, target_b=b, mix=mix)
    assert torch.equal(one, cross_entropy_hip(x, a, target_b=b, mix=mix.float()))
    assert torch.equal(cross_entropy_hip(x, a, target_b=b, mix=1), cross_entropy_hip(x, a))
    assert torch.equal(cross_entropy_hip(x, a, target_b=b, mix=0), cross_entropy_hip(x, b))
    assert torch.equal(cross_entropy_hip(x, a, label_smoothing=0), cross_entropy_hip(x, a))
    with pytest.raises(ValueError, match="target"):
        cross_entropy_hip(x, a.cpu())
    with pytest.raises(ValueError, match="mix"):
        cross_entropy_hip(x, a, target_b=b, mix=1.5)
    with pytest.raises(ValueError, match="post_weight"):
        block_norms_hip(x, x, post_weight=torch.ones(50))
    with pytest.raises(ValueError, match="eps"):
        rms_norm_hip(x, torch.ones(50, device=DEV), eps=-1)


def test_parameters_in_the_same_memory_are_refused() -> None:
    announce("adamw overlapping parameters")
    flat = torch.zeros(10000, device=DEV)
    p, q, r = (torch.nn.Parameter(flat[a:b]) for a, b in ((0, 5000), (5000, 10000), (4999, 6000)))
    for t in (p, q, r):
        t.grad = torch.ones_like(t)
    AdamW([p, q]).step()  # beside each other
    kept = flat.clone()
    with pytest.raises(ValueError, match="share memory"):
        AdamW([p, r]).step()
    assert torch.equal(flat, kept)


def test_a_master_copy_is_what_a_step_starts_from() -> None:
    announce("adamw master copy")
    p = torch.nn.Parameter(torch.ones(300, device=DEV).bfloat16())
    opt = AdamW([p], lr=0.0, weight_decay=0.0, master_weights=True)
    p.grad = torch.ones_like(p)
    opt.step()
    with torch.no_grad():
        p.fill_(2.0)
        opt.state[p]["master"].fill_(2.0)
    opt.step()
    assert (p == 2).all()
