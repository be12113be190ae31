"""Performance cases of the operators around the BiGEMM in a training step.

Three operators, each through the package's public entry points:

* ``norms``  ``block_norms_hip``: the norm after a block, its gate and residual scale, the residual, and
             the norm before the next block, as inference (``fwd``) or forward and backward (``train``);
             with ``delta`` false the norm before a block alone (``rms_norm_hip``);
* ``adamw``  ``AdamW.step``: one update of many parameters at once, with states in 32 or 8 bits, with or
             without fp32 master weights and clipping of the gradients' norm;
* ``xent``   ``cross_entropy_hip``: softmax cross-entropy, loss and gradient, with one label or two
             weighted ones per row, label smoothing and rows that are left out.

Where ``own`` is false, ``run`` computes the same by elementary torch operations in 32 bits.
"""

from __future__ import annotations

import math
import random

import torch

own = False
DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-6

WIDTHS, DEPTHS, TILES, CLASSES = (128, 256, 512, 1024), (2, 3, 8, 2), (64, 64, 128, 128), 1000
ANCHORED = (2, 3)  # stages (from 0) that begin with a Linear
G = 16  # tokens of a group

LR, BETA1, BETA2, ADAM_EPS, DECAY, MAX_NORM = 1e-3, 0.9, 0.999, 1e-8, 0.05, 1.0
BLOCK = 256      # values that share one scale of an 8-bit state
COUNTED = 4096   # values that share one step counter
SMALL = 4096     # smaller tensors hold 32-bit states under state_bits=8 too
FP8_MOST = 448.0  # largest e4m3fn value

IGNORED = -100

# Most values of a drawn case.
MOST_NORM_16BIT, MOST_NORM_F32 = 128 * 56 * 56 * 128, 32 * 28 * 28 * 256
MOST_PARAMS, MOST_LOGITS = 64 << 20, 4096 * 21841


def _norms(name, b, n, c, dtype, do, delta=True, post=True, gate="channel", scale=False, nxt=True, weights="same"):
    case = {"op": "norms", "do": do, "b": b, "n": n, "c": c, "dtype": dtype, "delta": delta, "post": post and delta,
            "gate": gate if delta else "none", "scale": scale and delta, "next": nxt and delta, "weights": weights}
    return {"name": name, **case} if name else case


def _adamw(name, layout, size, dtype, bits, master=False, clip=False, steps=100):
    case = {"op": "adamw", "layout": layout, "size": size, "dtype": dtype, "bits": bits, "master": master,
            "clip": clip, "steps": steps}
    return {"name": name, **case} if name else case


def _xent(name, rows, k, dtype, mixed=False, smoothing=0.0, left_out=0.0):
    case = {"op": "xent", "rows": rows, "k": k, "dtype": dtype, "mixed": mixed, "smoothing": smoothing,
            "left_out": left_out}
    return {"name": name, **case} if name else case


def listed():
    return [
        # One image through a late layer: the latency point of serving.
        _norms("norms_7x7x1024_b1_f16", 1, 49, 1024, "f16", "fwd"),
        # An early layer at full batch, the most activations of any layer: throughput inference.
        _norms("norms_56x56x128_b128_bf16", 128, 56 * 56, 128, "bf16", "fwd"),
        # Training the stage that most layers belong to, with drop-path.
        _norms("norms_train_14x14x512_b128_bf16", 128, 196, 512, "bf16", "train", scale=True, weights="f32"),
        # Training in the default dtype of a new model, the gate made for each image.
        _norms("norms_train_28x28x256_b32_f32", 32, 784, 256, "f32", "train", gate="image"),
        # A narrower network at 160 px whose channels fill no vector.
        _norms("norms_train_40x40x95_b64_bf16", 64, 1600, 95, "bf16", "train"),
        # A new head on a frozen network: one matrix and its bias.
        _adamw("adamw_head_f32", "head", 1, "f32", 32),
        # The whole network as created (fp32), the first step of a run.
        _adamw("adamw_model_f32", "model", 1, "f32", 32, steps=0),
        # The whole network in mixed precision: bf16 weights with fp32 masters, 8-bit states, clipped.
        _adamw("adamw_model_bf16_master_8bit_clip", "model", 1, "bf16", 8, master=True, clip=True),
        # A network of four times the widths, where the states' bytes matter most.
        _adamw("adamw_wide4_f32_8bit", "model", 4, "f32", 8),
        # A few images' labels: the smallest loss.
        _xent("xent_8x1000_bf16", 8, CLASSES, "bf16"),
        # A large batch with mixed labels and smoothing, logits in fp32.
        _xent("xent_1024x1000_f32_mixed", 1024, CLASSES, "f32", mixed=True, smoothing=0.1),
        # Dense labels over a large class list of odd length, some rows left out.
        _xent("xent_4096x21841_bf16", 4096, 21841, "bf16", smoothing=0.1, left_out=0.1),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choices(["norms", "adamw", "xent"], [50, 25, 25])[0]
    dtype = rng.choices(["bf16", "f16", "f32"], [50, 20, 30])[0]
    if op == "norms":
        c = rng.choice(WIDTHS) if rng.random() < 0.5 else _log_int(rng, 1, 8192)
        most = MOST_NORM_F32 if dtype == "f32" else MOST_NORM_16BIT
        n = _log_int(rng, 1, max(1, min(56 * 56, most // c)))
        b = _log_int(rng, 1, max(1, min(128, most // (n * c))))
        return _norms(None, b, n, c, dtype, rng.choice(["fwd", "train"]), delta=rng.random() < 0.85,
                      post=rng.random() < 0.8, gate=rng.choice(["none", "channel", "channel", "image"]),
                      scale=rng.random() < 0.4, nxt=rng.random() < 0.7, weights=rng.choice(["same", "f32"]))
    if op == "adamw":
        if rng.random() < 0.3:
            layout, size = "model", rng.choice([1, 2])
        else:
            layout, size = "random", _log_int(rng, 1, MOST_PARAMS)
        return _adamw(None, layout, size, dtype, rng.choice([32, 8]), master=dtype != "f32" and rng.random() < 0.6,
                      clip=rng.random() < 0.5, steps=rng.choice([0, 1, 10, 1000, 100000]))
    k = CLASSES if rng.random() < 0.3 else _log_int(rng, 2, 200000)
    rows = _log_int(rng, 1, max(1, min(32768, (MOST_LOGITS if dtype != "f32" else MOST_LOGITS // 2) // k)))
    return _xent(None, rows, k, dtype, mixed=rng.random() < 0.4, smoothing=rng.choice([0.0, 0.1]),
                 left_out=rng.choice([0.0, 0.0, 0.2]))


# ---------------------------------------------------------------------------------------
# Inputs


def _generator(seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    return gen


def _norms_inputs(case, seed):
    gen = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    wdtype = dtype if case["weights"] == "same" else torch.float32
    b, n, c = case["b"], case["n"], case["c"]

    def normal(scale=1.0):
        return (torch.randn(b, n, c, generator=gen, device=DEVICE) * scale).to(dtype)

    def around_one(*shape):
        return (torch.rand(shape, generator=gen, device=DEVICE) + 0.5).to(wdtype)

    s = {"x": normal(), "delta": normal(0.3) if case["delta"] else None,
         "post": around_one(c) if case["post"] else None, "gate": None, "scale": None,
         "next": around_one(c) if case["next"] or not case["delta"] else None, "dout": None, "dnext": None}
    if case["gate"] != "none":
        s["gate"] = around_one(c) if case["gate"] == "channel" else around_one(b, c)
    if case["scale"]:  # drop-path: images that are left out, the others scaled up
        s["scale"] = (torch.rand(b, generator=gen, device=DEVICE) >= 0.1).float() / 0.9
    if case["do"] == "train":
        s["dout"] = normal() if case["delta"] else None
        s["dnext"] = normal() if s["next"] is not None else None
    return s


def _shapes(case):
    """Shapes of the parameters, matrices and vectors as a network has them."""
    if case["layout"] == "head":
        return [(CLASSES, WIDTHS[3]), (CLASSES,)]
    if case["layout"] == "random":
        rng, left, shapes = random.Random(case["size"]), case["size"], []
        while left > 0 and len(shapes) < 200:
            n = left if len(shapes) == 199 else min(left, _log_int(rng, 1, max(1, left)))
            shapes.append((n,) if n % 2 or rng.random() < 0.4 else (2, n // 2))
            left -= n
        return shapes
    widths = [w * case["size"] for w in WIDTHS]
    shapes = [(widths[0], 48)] + [(widths[i + 1], 4 * widths[i]) for i in range(3)]
    for i in range(4):
        if i in ANCHORED:
            shapes.append((widths[i], widths[i]))
        d = TILES[i]
        q = widths[i] // d
        for _ in range(DEPTHS[i]):
            shapes += [(widths[i],), (G, G), (G, G), (G, G), (q, d, 2 * d), (q, d, 2 * d), (q, 2 * d, d), (widths[i],)]
    return shapes + [(CLASSES, widths[3]), (CLASSES,)]


def _places(case):
    """(shape, values, first value) of every parameter in one buffer, each at a whole block, the tensors with
    32-bit states first; the buffer's length and that of its 32-bit part."""
    items, at, split = [], 0, None
    few = SMALL if case["bits"] == 8 else 0
    shapes = _shapes(case)
    order = sorted(range(len(shapes)), key=lambda i: case["bits"] == 8 and math.prod(shapes[i]) >= few)
    for i in order:
        n = math.prod(shapes[i])
        if split is None and (case["bits"] == 8 and n >= few):
            split = at
        items.append((shapes[i], n, at))
        at += -(-n // BLOCK) * BLOCK
    return items, at, at if split is None else split


def _adamw_inputs(case, seed):
    """One buffer each for parameters, gradients, masters and states; padding between tensors is zero."""
    gen = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    items, total, split = _places(case)
    fill = torch.zeros(total // BLOCK, BLOCK, dtype=torch.bool)
    flat = fill.view(-1)
    decay = torch.zeros(total // BLOCK, 1)
    for shape, n, at in items:
        flat[at:at + n] = True
        decay[at // BLOCK: -(-(at + n) // BLOCK)] = DECAY if len(shape) > 1 else 0.0
    fill, decay = fill.to(DEVICE), decay.to(DEVICE)

    def normal(scale):
        return torch.randn(total // BLOCK, BLOCK, generator=gen, device=DEVICE) * scale * fill

    weights = normal(0.02)
    s = {"case": case, "items": items, "split": split // BLOCK, "t": case["steps"], "decay": decay,
         "p": weights.to(dtype), "master": weights if case["master"] else None, "g": normal(1e-3).to(dtype)}
    del weights, flat
    started = case["steps"] > 0
    m = normal(5e-4) if started else torch.zeros(total // BLOCK, BLOCK, device=DEVICE)
    # roots of the second moment between 1e-4 and 3e-3
    root = torch.exp(torch.rand(total // BLOCK, BLOCK, generator=gen, device=DEVICE) * 3.4 - 9.2) * fill
    root = root if started else torch.zeros_like(root)
    k = s["split"]
    s["m"], s["v"] = m[:k].clone(), root[:k].square()
    m8, root8 = m[k:], root[k:]
    s["m_scale"], s["v_scale"] = m8.abs().amax(1) / FP8_MOST, root8.amax(1) / FP8_MOST
    s["m8"] = (m8 / s["m_scale"].clamp(min=1e-30)[:, None]).clamp(-FP8_MOST, FP8_MOST).to(torch.float8_e4m3fn)
    s["v8"] = (root8 / s["v_scale"].clamp(min=1e-30)[:, None]).clamp(0, FP8_MOST).to(torch.float8_e4m3fn)
    return s


def _xent_inputs(case, seed):
    gen = _generator(seed)
    rows, k = case["rows"], case["k"]
    logits = (torch.randn(rows, k, generator=gen, device=DEVICE) * 3).to(DTYPES[case["dtype"]])

    def labels():
        return torch.randint(0, k, (rows,), generator=gen, device=DEVICE)

    a = labels()
    keep = torch.rand(rows, generator=gen, device=DEVICE) >= case["left_out"]
    keep[0] = True  # a batch with no label at all has no mean
    # fp16 gradients need a scaled loss to keep their small values.
    scale = 16.0 * rows if case["dtype"] == "f16" else 1.0
    return {"case": case, "logits": logits, "a": torch.where(keep, a, IGNORED), "b": labels() if case["mixed"] else None,
            "mix": torch.rand(rows, generator=gen, device=DEVICE) if case["mixed"] else None,
            "up": torch.full((), scale, device=DEVICE)}


def _optimizer(s):
    """The optimizer of the parameters in the buffers, with their states in the buffers too."""
    import omniwave_amd

    case, split = s["case"], s["split"]
    groups = ([], [])
    state = []
    for shape, n, at in s["items"]:
        p = torch.nn.Parameter(s["p"].view(-1)[at:at + n].view(shape))
        p.grad = s["g"].view(-1)[at:at + n].view(shape)
        groups[len(shape) == 1].append(p)
        first = at // BLOCK
        entry = {"step": torch.full((-(-n // COUNTED),), case["steps"], dtype=torch.int32, device=DEVICE)}
        if first < split:
            entry["exp_avg"] = s["m"].view(-1)[at:at + n].view(shape)
            entry["exp_avg_sq"] = s["v"].view(-1)[at:at + n].view(shape)
        else:
            first, off, blocks = first - split, at - split * BLOCK, -(-n // BLOCK)
            entry["exp_avg"] = s["m8"].view(-1)[off:off + n].view(shape)
            entry["exp_avg_sq_root"] = s["v8"].view(-1)[off:off + n].view(shape)
            entry["exp_avg_scale"] = s["m_scale"][first:first + blocks]
            entry["exp_avg_sq_root_scale"] = s["v_scale"][first:first + blocks]
        if s["master"] is not None:
            entry["master"] = s["master"].view(-1)[at:at + n].view(shape)
        state.append((p, entry))
    opt = omniwave_amd.AdamW(
        [{"params": ps, "weight_decay": wd} for ps, wd in zip(groups, (DECAY, 0.0)) if ps], lr=LR, betas=(BETA1, BETA2),
        eps=ADAM_EPS, state_bits=case["bits"], master_weights=case["master"],
        max_grad_norm=MAX_NORM if case["clip"] else None)
    for p, entry in state:
        opt.state[p] = entry
    return opt


def prepare(case, seed):
    if case["op"] == "norms":
        s = {"case": case, **_norms_inputs(case, seed)}
        if case["do"] == "train":
            for name in ("x", "delta", "post", "gate", "next"):
                if s[name] is not None:
                    s[name].requires_grad_(True)
        return s
    if case["op"] == "adamw":
        s = _adamw_inputs(case, seed)
        if own:
            s["optimizer"] = _optimizer(s)
        return s
    s = _xent_inputs(case, seed)
    s["logits"].requires_grad_(True)
    return s


# ---------------------------------------------------------------------------------------
# The plain forms


@torch.no_grad()
def _norms_plain(s):
    case, dtype = s["case"], s["x"].dtype
    x = s["x"].float()
    if not case["delta"]:
        w = s["next"].float()
        r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
        outs = {"next": (x * r * w).to(dtype)}
        if case["do"] == "train":
            g = s["dnext"].float()
            h = g * w
            outs["dx"] = (r * (h - x * (r * r) * (x * h).mean(-1, keepdim=True))).to(dtype)
            outs["dnext_weight"] = (g * x * r).sum((0, 1)).to(s["next"].dtype)
        return outs
    b = case["b"]
    delta = s["delta"].float()
    scale = 1.0 if s["scale"] is None else s["scale"].view(b, 1, 1)
    gate = 1.0
    if s["gate"] is not None:
        gate = s["gate"].float() if case["gate"] == "channel" else s["gate"].float()[:, None]
    p, r1 = delta, None
    if s["post"] is not None:
        r1 = torch.rsqrt(delta.square().mean(-1, keepdim=True) + EPS)
        p = delta * r1 * s["post"].float()
    out = x + scale * gate * p
    outs = {"out": out.to(dtype)}
    if s["next"] is not None:
        w2 = s["next"].float()
        r2 = torch.rsqrt(out.square().mean(-1, keepdim=True) + EPS)
        outs["next"] = (out * r2 * w2).to(dtype)
    if case["do"] != "train":
        return outs
    g = s["dout"].float()
    if s["next"] is not None:
        gn = s["dnext"].float()
        h = gn * w2
        g = g + r2 * (h - out * (r2 * r2) * (out * h).mean(-1, keepdim=True))
        outs["dnext_weight"] = (gn * out * r2).sum((0, 1)).to(s["next"].dtype)
    outs["dx"] = g.to(dtype)
    e = g * scale
    if s["gate"] is not None:
        outs["dgate"] = (e * p).sum((0, 1) if case["gate"] == "channel" else 1).to(s["gate"].dtype)
    q = e * gate
    if s["post"] is not None:
        outs["dpost_weight"] = (q * delta * r1).sum((0, 1)).to(s["post"].dtype)
        h = q * s["post"].float()
        q = r1 * (h - delta * (r1 * r1) * (delta * h).mean(-1, keepdim=True))
    outs["ddelta"] = q.to(dtype)
    return outs


def _to_fp8(values, scale):
    inv = torch.where(scale > 0, 1.0 / scale, 0.0)
    return (values * inv[:, None]).clamp(-FP8_MOST, FP8_MOST)


@torch.no_grad()
def _adamw_plain(s):
    case, k = s["case"], s["split"]
    s["t"] += 1
    t = s["t"]
    p = s["p"].float() if s["master"] is None else s["master"]
    g = s["g"].float()
    norm = None
    if case["clip"]:
        norm = g.double().square().sum().sqrt().float()
        g = g * torch.clamp(MAX_NORM / (norm + 1e-6), max=1.0)
    m = torch.cat([s["m"], s["m8"].float() * s["m_scale"][:, None]])
    v = torch.cat([s["v"], (s["v8"].float() * s["v_scale"][:, None]).square()])
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + g * g * (1 - BETA2)
    root = v.sqrt()
    step = LR / (1 - BETA1 ** t)
    p = p * (1 - LR * s["decay"]) - step * (m / (root * (1 / math.sqrt(1 - BETA2 ** t)) + ADAM_EPS))
    s["p"].copy_(p)
    if s["master"] is not None:
        s["master"].copy_(p)
    s["m"].copy_(m[:k])
    s["v"].copy_(v[:k])
    m8, root8 = m[k:], root[k:]
    s["m_scale"].copy_(m8.abs().amax(1) / FP8_MOST)
    s["v_scale"].copy_(root8.amax(1) / FP8_MOST)
    s["m8"].copy_(_to_fp8(m8, s["m_scale"]))
    least = torch.where(root8 > 0, 2.0 ** -9, 0.0)
    s["v8"].copy_(torch.maximum(_to_fp8(root8, s["v_scale"]), least))
    return _adamw_outputs(s, norm)


def _adamw_outputs(s, norm):
    """The updated parameters and states.  An 8-bit state is held as float8 values and the scale of every block."""
    outs = {"p": s["p"], "master": s["master"], "norm": norm}
    if s["m"].numel():
        outs.update(m=s["m"], v=s["v"])
    if s["m8"].numel():
        outs.update(m8=s["m8"], v8=s["v8"], m_scale=s["m_scale"], v_scale=s["v_scale"])
    return outs


@torch.no_grad()
def _xent_plain(s):
    eps, k = s["case"]["smoothing"], s["case"]["k"]
    x = s["logits"].float()
    valid = s["a"] != IGNORED
    a = torch.where(valid, s["a"], 0)[:, None]
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    z = e.sum(1, keepdim=True)
    lse = torch.log(z) + top
    picked = x.gather(1, a)
    mix = None
    if s["b"] is not None:
        mix = s["mix"][:, None]
        picked = mix * picked + (1 - mix) * x.gather(1, s["b"][:, None])
    losses = (1 - eps) * (lse - picked)
    if eps:
        losses = losses + eps * (lse - x.mean(1, keepdim=True))
    count = valid.sum()
    loss = torch.where(valid[:, None], losses, 0).sum() / count
    grad = e / z - eps / k
    grad.scatter_add_(1, a, -(1 - eps) * (torch.ones_like(lse) if mix is None else mix))
    if mix is not None:
        grad.scatter_add_(1, s["b"][:, None], -(1 - eps) * (1 - mix))
    grad = grad * (s["up"] / count) * valid[:, None]
    return {"loss": loss, "dlogits": grad.to(s["logits"].dtype)}


# ---------------------------------------------------------------------------------------
# The framework's operators


def _norms_own(s):
    import omniwave_amd

    case = s["case"]
    if not case["delta"]:
        if case["do"] == "fwd":
            with torch.inference_mode():
                return {"next": omniwave_amd.rms_norm_hip(s["x"], s["next"], eps=EPS)}
        nxt = omniwave_amd.rms_norm_hip(s["x"], s["next"], eps=EPS)
        dx, dw = torch.autograd.grad(nxt, (s["x"], s["next"]), s["dnext"])
        return {"next": nxt.detach(), "dx": dx, "dnext_weight": dw}
    args = dict(post_weight=s["post"], gate=s["gate"], scale=s["scale"], next_weight=s["next"], eps=EPS)
    if case["do"] == "fwd":
        with torch.inference_mode():
            out, nxt = omniwave_amd.block_norms_hip(s["x"], s["delta"], **args)
        return {"out": out, "next": nxt}
    out, nxt = omniwave_amd.block_norms_hip(s["x"], s["delta"], **args)
    leaves = {"dx": s["x"], "ddelta": s["delta"], "dpost_weight": s["post"], "dgate": s["gate"], "dnext_weight": s["next"]}
    leaves = {name: t for name, t in leaves.items() if t is not None}
    outs = (out,) if nxt is None else (out, nxt)
    grads = torch.autograd.grad(outs, tuple(leaves.values()), (s["dout"], s["dnext"])[:len(outs)])
    return {"out": out.detach(), "next": None if nxt is None else nxt.detach(), **dict(zip(leaves, grads))}


def _adamw_own(s):
    s["optimizer"].step()
    return _adamw_outputs(s, s["optimizer"].grad_norm)


def _xent_own(s):
    import omniwave_amd

    loss = omniwave_amd.cross_entropy_hip(s["logits"], s["a"], target_b=s["b"], mix=s["mix"],
                                          label_smoothing=s["case"]["smoothing"], ignore_index=IGNORED)
    (grad,) = torch.autograd.grad(loss, s["logits"], s["up"])
    return {"loss": loss.detach(), "dlogits": grad}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norms": _norms_own, "adamw": _adamw_own, "xent": _xent_own}[op](state)
    return {"norms": _norms_plain, "adamw": _adamw_plain, "xent": _xent_plain}[op](state)


# ---------------------------------------------------------------------------------------
# Work


def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "norms":
        values = case["b"] * case["n"] * case["c"]
        train = case["do"] == "train"
        tensors = 2 + case["delta"] + (case["next"] if case["delta"] else 0)  # in: x, delta; out: out, next
        flops = 10.0
        if train:  # in: dout, dnext; out: dx, ddelta
            tensors += 2 if not case["delta"] else 3 + case["next"]
            flops = 35.0
        wsize = 4 if case["weights"] == "f32" else size
        vectors = case["post"] + (case["next"] or not case["delta"])
        weights = case["c"] * (vectors + {"none": 0, "channel": 1, "image": case["b"]}[case["gate"]])
        return {"bytes": float(tensors * values * size + weights * wsize * (2 if train else 1)), "flops": flops * values}
    if case["op"] == "adamw":
        total = few = 0
        for shape in _shapes(case):
            n = math.prod(shape)
            total += n
            few += n if case["bits"] == 32 or n < SMALL else 0
        moved = total * (size + (8 + size if case["master"] else 2 * size)) + 16 * few
        moved += (total - few) * (4 + 16 / BLOCK)
        return {"bytes": float(moved), "flops": 20.0 * total}
    values = case["rows"] * case["k"]
    return {"bytes": float(2 * values * size + case["rows"] * (20 if case["mixed"] else 8)), "flops": 8.0 * values}


# ---------------------------------------------------------------------------------------
# The same results in 64 bits


def _unit(t):
    """Rows of root mean square one."""
    return t / (torch.linalg.vector_norm(t, dim=-1, keepdim=True).square() / t.shape[-1] + EPS).sqrt()


def _norms_exact(case, seed):
    s = _norms_inputs(case, seed)
    train = case["do"] == "train"
    v = {k: s[k].double().requires_grad_(train) for k in ("x", "delta", "post", "gate", "next") if s[k] is not None}
    out = v["x"]
    if case["delta"]:
        branch = _unit(v["delta"]) * v["post"] if "post" in v else v["delta"]
        if "gate" in v:
            branch = branch * (v["gate"][:, None] if case["gate"] == "image" else v["gate"])
        if s["scale"] is not None:
            branch = branch * s["scale"].double()[:, None, None]
        out = out + branch
    result = {"out": out} if case["delta"] else {}
    if "next" in v:
        result["next"] = _unit(out) * v["next"]
    if train:
        ups = [s["dout"] if name == "out" else s["dnext"] for name in result]
        loss = sum((t * u.double()).sum() for t, u in zip(result.values(), ups))
        names = {"x": "dx", "delta": "ddelta", "post": "dpost_weight", "gate": "dgate", "next": "dnext_weight"}
        result.update(zip((names[k] for k in v), torch.autograd.grad(loss, tuple(v.values()))))
    return {k: t.detach() for k, t in result.items()}


def _nearest_fp8(y):
    """The nearest e4m3fn value, ties to the even one: eight steps to an octave, 2^-9 apart below 2^-6."""
    _, exponent = torch.frexp(y)
    step = torch.ldexp(torch.ones_like(y), torch.clamp(exponent - 4, min=-9))
    return torch.round(y / step) * step


def _adamw_exact(case, seed):
    s = _adamw_inputs(case, seed)
    k, t = s["split"], case["steps"] + 1
    p = (s["p"] if s["master"] is None else s["master"]).double()
    g = s["g"].double()
    norm = torch.linalg.vector_norm(g) if case["clip"] else None
    if case["clip"]:
        g *= min(1.0, MAX_NORM / (float(norm) + 1e-6))
    m = torch.lerp(g, torch.cat([s["m"].double(), s["m8"].double() * s["m_scale"].double()[:, None]]), BETA1)
    v = torch.cat([s["v"].double(), (s["v8"].double() * s["v_scale"].double()[:, None]) ** 2])
    v = torch.lerp(g * g, v, BETA2)
    p = p - LR * s["decay"].double() * p
    p -= LR * (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + ADAM_EPS)
    result = {"p": p, "master": None if s["master"] is None else p, "norm": norm}
    if k:
        result.update(m=m[:k], v=v[:k])
    if k < len(m):
        m8, root8 = m[k:], v[k:].sqrt()
        # The scale is part of the format: a 32-bit number.
        ms, vs = (m8.abs().amax(1) / FP8_MOST).float().double(), (root8.amax(1) / FP8_MOST).float().double()
        code = _nearest_fp8(root8 / vs.clamp(min=1e-300)[:, None]).clamp(max=FP8_MOST)
        code = torch.where((root8 > 0) & (code < 2.0 ** -9), 2.0 ** -9, code)
        result.update(m8=_nearest_fp8(m8 / ms.clamp(min=1e-300)[:, None]).clamp(-FP8_MOST, FP8_MOST), v8=code,
                      m_scale=ms, v_scale=vs)
    return result


def _xent_exact(case, seed):
    s = _xent_inputs(case, seed)
    rows, k, eps = case["rows"], case["k"], case["smoothing"]
    left = s["a"] != IGNORED
    count = int(left.sum())
    up, loss, grads = float(s["up"]), 0.0, torch.zeros(rows, k, dtype=torch.float64, device=DEVICE)
    for part in torch.arange(rows, device=DEVICE).split(max(1, 50_000_000 // k)):
        part = part[left[part]]
        if not len(part):
            continue
        x = s["logits"][part].double().requires_grad_(True)
        want = torch.full_like(x, eps / k).detach()
        one = torch.nn.functional.one_hot
        w = torch.ones(len(part), 1, dtype=torch.float64, device=DEVICE) if s["mix"] is None else s["mix"][part].double()[:, None]
        want += (1 - eps) * w * one(s["a"][part], k)
        if s["b"] is not None:
            want += (1 - eps) * (1 - w) * one(s["b"][part], k)
        value = -(want * torch.log_softmax(x, 1)).sum() / count
        grads[part] = torch.autograd.grad(value * up, x)[0]
        loss += float(value)
    return {"loss": torch.tensor(loss, dtype=torch.float64), "dlogits": grads}


def exact(case, seed):
    return {"norms": _norms_exact, "adamw": _adamw_exact, "xent": _xent_exact}[case["op"]](case, seed)
