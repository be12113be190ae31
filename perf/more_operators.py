"""Performance cases of layer norm, the gated feed-forward product and distillation.

Three operators, each through the package's public entry points:

* ``lnorm``    ``layer_norm_hip``: layer norm of rows, as inference (``fwd``) or forward and backward (``train``);
* ``gated``    ``gated_linear_hip``: both projections of a gated feed-forward block, SiLU of the one and their
               product, ``fwd`` or ``train``;
* ``distill``  ``distillation_hip``: loss against a teacher's top logits, with its gradient.

Where ``own`` is false, ``run`` computes the same by elementary torch operations in 32 bits.
"""

from __future__ import annotations

import math

import torch

own = False
DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-6
WIDTHS, CLASSES = (128, 256, 512, 1024), 1000
ABSENT = -100  # index of an entry that a teacher's list does not have

# Most values (products) of a drawn case.
MOST_NORM_16BIT, MOST_NORM_F32 = 128 * 56 * 56 * 128, 32 * 28 * 28 * 256
MOST_GATED_VALUES, MOST_GATED_16BIT, MOST_GATED_F32 = 128 * 56 * 56 * 256, 6272 * 4096 * 8192, 25088 * 1024 * 512
MOST_LOGITS = 4096 * 21841


def _lnorm(name, rows, c, dtype, do, weight=True, bias=True, weights="same"):
    case = {"op": "lnorm", "do": do, "rows": rows, "c": c, "dtype": dtype, "weight": weight, "bias": bias,
            "weights": weights}
    return {"name": name, **case} if name else case


def _gated(name, rows, c, hidden, dtype, do):
    case = {"op": "gated", "do": do, "rows": rows, "c": c, "hidden": hidden, "dtype": dtype}
    return {"name": name, **case} if name else case


def _distill(name, rows, k, top, dtype, temperature, absent=0.0, empty=0.0):
    case = {"op": "distill", "rows": rows, "k": k, "top": top, "dtype": dtype, "temperature": temperature,
            "absent": absent, "empty": empty}
    return {"name": name, **case} if name else case


def listed():
    return [
        # The pooled features of one image before the head: the latency point of serving.
        _lnorm("lnorm_1x1024_f16", 1, 1024, "f16", "fwd"),
        # An early layer at full batch, the most activations of any layer: throughput inference.
        _lnorm("lnorm_56x56x128_b128_bf16", 128 * 56 * 56, 128, "bf16", "fwd"),
        # Training the stage that most layers belong to, weights kept in fp32.
        _lnorm("lnorm_train_14x14x512_b128_bf16", 128 * 196, 512, "bf16", "train", weights="f32"),
        # A narrower network at 160 px whose channels fill no vector, in the default dtype of a new model.
        _lnorm("lnorm_train_40x40x95_b64_f32", 64 * 1600, 95, "f32", "train"),
        # One token through the widest layer: serving's smallest call, bound by reading the weights.
        _gated("gated_1x1024_f16", 1, 1024, 2048, "f16", "fwd"),
        # One image's tokens through the last stage.
        _gated("gated_7x7x1024_b1_bf16", 49, 1024, 2048, "bf16", "fwd"),
        # The first stage at full batch: many tokens, few channels.
        _gated("gated_train_56x56x128_b128_bf16", 128 * 56 * 56, 128, 256, "bf16", "train"),
        # The second stage in the default dtype of a new model.
        _gated("gated_train_28x28x256_b32_f32", 32 * 784, 256, 512, "f32", "train"),
        # A network of four times the widths, the last stage: large products.
        _gated("gated_train_7x7x4096_b128_bf16", 128 * 49, 4096, 8192, "bf16", "train"),
        # A few images: the smallest loss.
        _distill("distill_8x1000_top8_bf16", 8, CLASSES, 8, "bf16", 2.0),
        # A large batch, lists of several lengths, logits in fp32.
        _distill("distill_1024x1000_top100_f32", 1024, CLASSES, 100, "f32", 1.0, absent=0.2),
        # Dense predictions over a large class list of odd length, some rows without a teacher.
        _distill("distill_4096x21841_top64_bf16", 4096, 21841, 64, "bf16", 4.0, empty=0.1),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["lnorm", "gated", "gated", "distill"])
    dtype = rng.choices(["bf16", "f16", "f32"], [50, 20, 30])[0]
    do = rng.choice(["fwd", "train"])
    if op == "lnorm":
        c = rng.choice(WIDTHS) if rng.random() < 0.4 else _log_int(rng, 8, 8192)
        rows = _log_int(rng, 1, max(1, (MOST_NORM_F32 if dtype == "f32" else MOST_NORM_16BIT) // max(c, 32)))
        return _lnorm(None, rows, c, dtype, do, weight=rng.random() < 0.9, bias=rng.random() < 0.7,
                      weights=rng.choice(["same", "f32"]))
    if op == "gated":
        c = rng.choice(WIDTHS) if rng.random() < 0.5 else _log_int(rng, 8, 4096)
        hidden = rng.choice([2, 4]) * c if rng.random() < 0.6 else _log_int(rng, 8, 8192)
        products = (MOST_GATED_F32 if dtype == "f32" else MOST_GATED_16BIT) // (c * hidden)
        rows = _log_int(rng, 1, max(1, min(128 * 56 * 56, products, MOST_GATED_VALUES // max(c, hidden))))
        return _gated(None, rows, c, hidden, dtype, do)
    k = CLASSES if rng.random() < 0.3 else _log_int(rng, 2, 200000)
    rows = _log_int(rng, 1, max(1, min(32768, (MOST_LOGITS if dtype != "f32" else MOST_LOGITS // 2) // k)))
    return _distill(None, rows, k, _log_int(rng, 1, min(k, 512)), dtype, rng.choice([1.0, 2.0, 4.0, 0.7]),
                    absent=rng.choice([0.0, 0.3]), empty=rng.choice([0.0, 0.0, 0.2]))


# ---------------------------------------------------------------------------------------
# Inputs


def _generator(seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    return gen


def _lnorm_inputs(case, seed):
    gen = _generator(seed)
    dtype, rows, c = DTYPES[case["dtype"]], case["rows"], case["c"]
    wdtype = dtype if case["weights"] == "same" else torch.float32
    # Channels have means and scales of their own, as activations do.
    mean = torch.randn(c, generator=gen, device=DEVICE)
    x = (torch.randn(rows, c, generator=gen, device=DEVICE) + 0.5 * mean).to(dtype)
    weight = (torch.rand(c, generator=gen, device=DEVICE) + 0.5).to(wdtype)
    bias = (torch.randn(c, generator=gen, device=DEVICE) * 0.1).to(wdtype)
    up = torch.randn(rows, c, generator=gen, device=DEVICE).to(dtype)
    return {"x": x, "weight": weight if case["weight"] else None, "bias": bias if case["bias"] else None,
            "up": up if case["do"] == "train" else None}


def _gated_inputs(case, seed):
    gen = _generator(seed)
    dtype, rows, c, hidden = DTYPES[case["dtype"]], case["rows"], case["c"], case["hidden"]

    def normal(n, k, scale):
        return (torch.randn(n, k, generator=gen, device=DEVICE) * scale).to(dtype)

    # Tokens behind a norm; projections that keep the scale.
    s = {"x": normal(rows, c, 1.0), "gate": normal(hidden, c, c ** -0.5), "up": normal(hidden, c, c ** -0.5)}
    s["dh"] = normal(rows, hidden, 0.1) if case["do"] == "train" else None
    return s


def _distill_inputs(case, seed):
    gen = _generator(seed)
    rows, k, top, dtype = case["rows"], case["k"], case["top"], DTYPES[case["dtype"]]
    teacher = torch.randn(rows, k, generator=gen, device=DEVICE) * 3
    # A student on its way to the teacher.
    student = (0.6 * teacher + 2.4 * torch.randn(rows, k, generator=gen, device=DEVICE)).to(dtype)
    values, indices = teacher.topk(top, 1)
    gone = torch.rand(rows, top, generator=gen, device=DEVICE) < case["absent"]
    gone |= torch.rand(rows, 1, generator=gen, device=DEVICE) < case["empty"]
    gone[0] = False  # a batch without any teacher has no mean
    # fp16 gradients need a scaled loss to keep their small values.
    scale = 16.0 * rows if case["dtype"] == "f16" else 1.0
    return {"logits": student, "values": values.to(dtype), "indices": torch.where(gone, ABSENT, indices),
            "up": torch.full((), scale, device=DEVICE)}


_INPUTS = {"lnorm": _lnorm_inputs, "gated": _gated_inputs, "distill": _distill_inputs}


def prepare(case, seed):
    s = {"case": case, **_INPUTS[case["op"]](case, seed)}
    if case["op"] == "distill":
        s["logits"].requires_grad_(True)
    elif case["do"] == "train":
        leaves = [s["x"], s["weight"], s["bias"]] if case["op"] == "lnorm" else [s["x"], s["gate"], s["up"]]
        for t in leaves:
            if t is not None:
                t.requires_grad_(True)
    return s


# ---------------------------------------------------------------------------------------
# The plain forms


@torch.no_grad()
def _lnorm_plain(s):
    dtype, x = s["x"].dtype, s["x"].float()
    w = 1.0 if s["weight"] is None else s["weight"].float()
    x = x - x.mean(1, keepdim=True)
    r = torch.rsqrt(x.square().mean(1, keepdim=True) + EPS)
    n = x * r
    y = n * w if s["bias"] is None else n * w + s["bias"].float()
    outs = {"y": y.to(dtype)}
    if s["up"] is not None:
        g = s["up"].float()
        h = g * w
        outs["dx"] = (r * (h - h.mean(1, keepdim=True) - n * (h * n).mean(1, keepdim=True))).to(dtype)
        if s["weight"] is not None:
            outs["dweight"] = (g * n).sum(0).to(s["weight"].dtype)
        if s["bias"] is not None:
            outs["dbias"] = g.sum(0).to(s["bias"].dtype)
    return outs


@torch.no_grad()
def _gated_plain(s):
    dtype, x, wg, wu = s["x"].dtype, s["x"].float(), s["gate"].float(), s["up"].float()
    g, u = x @ wg.t(), x @ wu.t()
    sig = 1 / (1 + torch.exp(-g))
    outs = {"h": (g * sig * u).to(dtype)}
    if s["dh"] is not None:
        dh = s["dh"].float()
        du = dh * g * sig
        dg = dh * u * sig * (1 + g * (1 - sig))
        outs.update(dx=(dg @ wg + du @ wu).to(dtype), dgate=(dg.t() @ x).to(dtype), dup=(du.t() @ x).to(dtype))
    return outs


@torch.no_grad()
def _distill_plain(s):
    temp = s["case"]["temperature"]
    x = s["logits"].float() / temp
    here = s["indices"] != ABSENT
    at = torch.where(here, s["indices"], 0)
    t = torch.where(here, s["values"].float() / temp, -math.inf)
    some = here.any(1, keepdim=True)
    t = torch.where(some, t - t.amax(1, keepdim=True), 0)
    e = torch.where(here, torch.exp(t), 0)
    zt = torch.where(some, e.sum(1, keepdim=True), 1)
    q = e / zt
    x = x - x.amax(1, keepdim=True)
    p = torch.exp(x)
    z = p.sum(1, keepdim=True)
    p = p / z
    terms = torch.where(here, q * (t - torch.log(zt) - x.gather(1, at) + torch.log(z)), 0)
    count = some.sum()
    loss = temp * temp * terms.sum() / count
    grad = (p * some).scatter_add_(1, at, -q) * (s["up"] * temp / count)
    return {"loss": loss, "dlogits": grad.to(s["logits"].dtype)}


# ---------------------------------------------------------------------------------------
# The framework's operators


def _lnorm_own(s):
    import omniwave_amd

    if s["up"] is None:
        with torch.inference_mode():
            return {"y": omniwave_amd.layer_norm_hip(s["x"], s["weight"], s["bias"], eps=EPS)}
    y = omniwave_amd.layer_norm_hip(s["x"], s["weight"], s["bias"], eps=EPS)
    leaves = {"dx": s["x"], "dweight": s["weight"], "dbias": s["bias"]}
    leaves = {name: t for name, t in leaves.items() if t is not None}
    return {"y": y.detach(), **dict(zip(leaves, torch.autograd.grad(y, tuple(leaves.values()), s["up"])))}


def _gated_own(s):
    import omniwave_amd

    if s["dh"] is None:
        with torch.inference_mode():
            return {"h": omniwave_amd.gated_linear_hip(s["x"], s["gate"], s["up"])}
    h = omniwave_amd.gated_linear_hip(s["x"], s["gate"], s["up"])
    dx, dgate, dup = torch.autograd.grad(h, (s["x"], s["gate"], s["up"]), s["dh"])
    return {"h": h.detach(), "dx": dx, "dgate": dgate, "dup": dup}


def _distill_own(s):
    import omniwave_amd

    loss = omniwave_amd.distillation_hip(s["logits"], s["values"], s["indices"], temperature=s["case"]["temperature"],
                                         ignore_index=ABSENT)
    (grad,) = torch.autograd.grad(loss, s["logits"], s["up"])
    return {"loss": loss.detach(), "dlogits": grad}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"lnorm": _lnorm_own, "gated": _gated_own, "distill": _distill_own}[op](state)
    return {"lnorm": _lnorm_plain, "gated": _gated_plain, "distill": _distill_plain}[op](state)


# ---------------------------------------------------------------------------------------
# Work


def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "distill":
        values = case["rows"] * case["k"]
        return {"bytes": float(2 * values * size + case["rows"] * case["top"] * (8 + size)), "flops": 8.0 * values}
    train = case["do"] == "train"
    rows, c = case["rows"], case["c"]
    if case["op"] == "lnorm":  # in: x, the upstream gradient; out: y, dx
        wsize = 4 if case["weights"] == "f32" else size
        weights = c * (case["weight"] + case["bias"]) * wsize
        return {"bytes": float((4 if train else 2) * rows * c * size + (2 if train else 1) * weights),
                "flops": (25.0 if train else 8.0) * rows * c}
    tokens, weights = rows * (c + case["hidden"]), 2 * c * case["hidden"]  # x and h (dx and dh)
    return {"bytes": float((2 if train else 1) * (tokens + weights) * size),
            "flops": (12.0 if train else 4.0) * rows * c * case["hidden"]}


# ---------------------------------------------------------------------------------------
# The same results in 64 bits


def _lnorm_exact(case, seed):
    s = _lnorm_inputs(case, seed)
    train = case["do"] == "train"
    v = {k: s[k].double().requires_grad_(train) for k in ("x", "weight", "bias") if s[k] is not None}
    var, mean = torch.var_mean(v["x"], dim=-1, keepdim=True, correction=0)
    y = (v["x"] - mean) / (var + EPS).sqrt()
    if "weight" in v:
        y = y * v["weight"]
    if "bias" in v:
        y = y + v["bias"]
    result = {"y": y}
    if train:
        names = {"x": "dx", "weight": "dweight", "bias": "dbias"}
        grads = torch.autograd.grad((y * s["up"].double()).sum(), tuple(v.values()))
        result.update(zip((names[k] for k in v), grads))
    return {k: t.detach() for k, t in result.items()}


def _gated_exact(case, seed):
    s = _gated_inputs(case, seed)
    x, gate, up = s["x"].double(), s["gate"].double(), s["up"].double()
    g, u = torch.mm(x, gate.T), torch.mm(x, up.T)
    sig = torch.special.expit(g)
    act = g * sig
    result = {"h": act * u}
    if s["dh"] is not None:
        du = s["dh"].double()
        dg = du * u * (sig + act * (1 - sig))
        du = du * act
        result["dx"] = torch.addmm(torch.mm(dg, gate), du, up)
        result["dgate"], result["dup"] = torch.mm(dg.T, x), torch.mm(du.T, x)
    return result


def _distill_exact(case, seed):
    s = _distill_inputs(case, seed)
    rows, k, temp = case["rows"], case["k"], case["temperature"]
    here = s["indices"] != ABSENT
    taught = here.any(1)
    count = int(taught.sum())
    loss, grads = 0.0, torch.zeros(rows, k, dtype=torch.float64, device=DEVICE)
    for part in torch.arange(rows, device=DEVICE).split(max(1, 50_000_000 // k)):
        part = part[taught[part]]
        if not len(part):
            continue
        x = s["logits"][part].double().requires_grad_(True)
        scores = (s["values"][part].double() / temp).masked_fill(~here[part], -math.inf)
        log_q = torch.log_softmax(scores, 1)
        log_p = torch.log_softmax(x / temp, 1).gather(1, s["indices"][part].clamp(min=0))
        q = log_q.exp()
        value = temp ** 2 * (q * (log_q - log_p)).masked_fill(~here[part], 0.0).sum() / count
        grads[part] = torch.autograd.grad(value * float(s["up"]), x)[0]
        loss += float(value.detach())
    return {"loss": torch.tensor(loss, dtype=torch.float64), "dlogits": grads}


def exact(case, seed):
    return {"lnorm": _lnorm_exact, "gated": _gated_exact, "distill": _distill_exact}[case["op"]](case, seed)
