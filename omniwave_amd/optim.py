"""AdamW over all parameters of a model at once, as HIP kernels (``adamw.hip``).

``AdamW`` is a ``torch.optim.Optimizer`` (the reference trains with ``torch.optim.AdamW``, a clip of the
gradients' norm and a check that it is finite, omniweave/training/engine.py:204-258): one launch updates as
many tensors as fit in a kernel's arguments, the clip needs one more, and nothing waits for the device, so
a step can be captured into a HIP graph.
"""

from __future__ import annotations

import ctypes
import math
from itertools import chain, groupby
from operator import is_

import numpy as np
import torch
from torch import Tensor
from torch.optim import optimizer as _base

from omniwave_amd import _native
from omniwave_amd.hip import _DTYPE_CODE, SUPPORTED_DTYPES, _stream_ptr
from omniwave_amd.norms import gpu_reason

CHUNK, BLOCK = _native.OW_ADAMW_CHUNK, _native.OW_ADAMW_BLOCK
FP8 = torch.float8_e4m3fn
FP8_MOST = 448.0
MIN_8BIT_VALUES = 4096  # smaller tensors keep 32-bit states: their bytes do not matter, their errors do
# Options of torch.optim.AdamW's groups that make another update, with the values that do not.
_PLAIN_UPDATE = {"maximize": False, "amsgrad": False, "differentiable": False, "decoupled_weight_decay": True}
_GRAD = 1  # field of OwAdamwTensor, whose fields are 8 bytes each
# Whether torch has the names by which a step sees that nothing listens to it; without them the base class wraps it.
_SHORTCUT = (hasattr(_base, "_global_optimizer_pre_hooks") and hasattr(_base, "_global_optimizer_post_hooks")
             and hasattr(torch.optim.Optimizer, "profile_hook_step")
             and hasattr(torch.autograd.profiler, "_is_profiler_enabled"))


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def _encode(values: Tensor, least: bool) -> tuple[Tensor, Tensor]:
    """fp32 values as e4m3fn and a scale per block (``least``: what is above zero stays above zero)."""
    flat = values.detach().float().reshape(-1)
    n = flat.numel()
    rows = torch.nn.functional.pad(flat, (0, -n % BLOCK)).reshape(-1, BLOCK)
    scale = rows.abs().amax(1) / FP8_MOST
    scale = torch.where(scale < torch.finfo(torch.float32).tiny, 0.0, scale)
    inv = torch.where(scale > 0, 1.0 / scale, 0.0)
    codes = (rows * inv[:, None]).clamp(-FP8_MOST, FP8_MOST).to(FP8)
    if least:
        codes = torch.where((rows > 0) & (codes.float() == 0), 2.0 ** -9, codes.float()).to(FP8)
    return codes.reshape(-1)[:n].reshape(values.shape), scale


def _decode(codes: Tensor, scale: Tensor) -> Tensor:
    flat = codes.float().reshape(-1)
    return (flat * scale.repeat_interleave(BLOCK)[:flat.numel()]).reshape(codes.shape)


class AdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW`` on the framework's kernels.

    ``state_bits``: 32, or 8 for states of tensors of at least 4,096 values in e4m3fn with an fp32 scale
    for every 256 values (the second moment as its root; see below what that costs).  ``master_weights``: keep
    fp32 copies of bf16 / fp16 parameters and update those, so that updates smaller than a parameter's rounding
    step are not lost.  ``max_grad_norm``: scale the gradients of each step so that their norm over all parameters is
    at most this, and skip the step (parameters, states and counters) where the norm is not finite;
    ``grad_norm`` is then the last step's norm, on the device (0 where nothing had a gradient; replays of a captured
    step write the tensor that it had at the capture).

    Parameters: contiguous, of fp32, bf16 or fp16, on one gfx950 GPU, no two in the same memory; gradients of
    the same dtype, dense.  With ``master_weights`` a step starts from the fp32 copy: a parameter that is
    changed otherwise (weights loaded or averaged in) has ``state[p]["master"]`` to be changed alike.
    ``lr`` may be a 0-dim fp32 tensor on the GPU, which a captured step reads anew; other
    hyperparameters of a captured step are those of its capture.  States are made by the first step, which
    therefore is not captured.  A step raises the parameters' version counters; the replay of a captured one
    cannot, so before an eager forward that follows replays call ``omniwave_amd.hip.clear_pack_cache()``.

    8-bit states save memory, not steps: they are the nearest codes after each step, and half a code's step is 3 to
    6% where a step moves the root of the second moment by 0.05% (beta2 = 0.999).  A change that a block of 256
    values shares is followed by the block's scale.  A change beside the block's largest value is not, but for
    gradients above some 8 times the root: where gradients fall tenfold beside a steady one the root stays up to
    tenfold too large (7.6 times in the median: steps too small), where they rise fourfold it reaches 0.4 to 1 of
    the right one (steps up to 2.6 times too large); where nothing changes it is 0.7 to 1.5 times the right one.
    A gradient that is not finite makes its block's states so, where 32-bit states lose one value
    (``max_grad_norm`` skips the step).

    ``state[p]``: ``step`` (int32, the steps done, one for every 4,096 values), ``exp_avg`` and
    ``exp_avg_sq`` (fp32), or ``exp_avg`` and ``exp_avg_sq_root`` (e4m3fn) with ``exp_avg_scale`` and
    ``exp_avg_sq_root_scale``, and ``master``.  ``load_state_dict`` also takes the states of
    ``torch.optim.AdamW`` and those of another ``state_bits``.  Groups and saved groups with ``maximize``, ``amsgrad``
    or ``differentiable``, or without ``decoupled_weight_decay``, are refused: their update is another one.
    """

    grad_norm: Tensor | None = None
    _plan: _Plan | None = None

    def __init__(self, params, lr: float | Tensor = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, state_bits: int = 32, master_weights: bool = False,
                 max_grad_norm: float | None = None) -> None:
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits!r}")
        if max_grad_norm is not None and not (max_grad_norm > 0 and math.isfinite(max_grad_norm)):
            raise ValueError(f"max_grad_norm must be positive and finite, got {max_grad_norm!r}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        self.state_bits, self.master_weights, self.max_grad_norm = state_bits, bool(master_weights), max_grad_norm

    def add_param_group(self, param_group: dict) -> None:
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            _hyper(group)
            if len(set(group["params"])) != len(group["params"]):
                raise ValueError("a parameter is in its group twice")
            for p in group["params"]:
                _check_parameter(p)
        except ValueError:
            self.param_groups.pop()
            raise
        self._plan = None

    def __getstate__(self) -> dict:
        kept = {k: getattr(self, k) for k in ("state_bits", "master_weights", "max_grad_norm")}
        return {**super().__getstate__(), **kept}

    # -- states ---------------------------------------------------------------------------

    def _layout(self, p: Tensor) -> dict[str, tuple[torch.dtype, tuple]]:
        """Names, dtypes and shapes of ``p``'s states."""
        n = p.numel()
        entry: dict[str, tuple[torch.dtype, tuple]] = {"step": (torch.int32, (-(-n // CHUNK),))}
        if self.state_bits == 8 and n >= MIN_8BIT_VALUES:
            scales = (torch.float32, (_blocks(n),))
            entry.update(exp_avg=(FP8, p.shape), exp_avg_sq_root=(FP8, p.shape), exp_avg_scale=scales,
                         exp_avg_sq_root_scale=scales)
        else:
            entry.update(exp_avg=(torch.float32, p.shape), exp_avg_sq=(torch.float32, p.shape))
        if self.master_weights and p.dtype != torch.float32:
            entry["master"] = (torch.float32, p.shape)
        return entry

    def _first_state(self, p: Tensor) -> None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW makes its states in the first step of a parameter, which cannot be captured: "
                               "run one step before the capture")
        entry = self.state[p]
        for name, (dtype, shape) in self._layout(p).items():
            if name == "master":
                entry[name] = p.detach().float()
            else:
                entry[name] = torch.zeros(shape, dtype=torch.uint8 if dtype == FP8 else dtype, device=p.device)
                if dtype == FP8:
                    entry[name] = entry[name].view(FP8)

    def _check_state(self, p: Tensor, layout: dict | None = None) -> None:
        entry, device = self.state[p], p.device
        for name, (dtype, shape) in (self._layout(p) if layout is None else layout).items():
            t = entry.get(name)
            if not isinstance(t, Tensor) or t.dtype != dtype or t.shape != shape or t.device != device \
                    or not t.is_contiguous():
                got = f"{t.dtype} {tuple(t.shape)} on {t.device}" if isinstance(t, Tensor) else repr(t)
                raise ValueError(f"state {name!r} of a parameter of shape {tuple(p.shape)} must be {dtype} {tuple(shape)}, "
                                 f"contiguous on {device}; got {got}")

    def load_state_dict(self, state_dict: dict) -> None:
        """``torch.optim.Optimizer.load_state_dict``; states keep their own dtypes, and those of
        ``torch.optim.AdamW`` or another ``state_bits`` are converted.  A dictionary that is refused changes nothing."""
        adopted: dict[Tensor, dict] = {}

        def before(_opt, loaded: dict) -> dict:  # behind the other hooks: this is what is loaded
            for group in loaded["param_groups"]:
                _refuse_other_updates(group)
            saved = dict(loaded["state"])
            ids = chain.from_iterable(g["params"] for g in loaded["param_groups"])
            params = chain.from_iterable(g["params"] for g in self.param_groups)
            # The base class would cast the states to the parameters' dtypes, a second set of them.
            adopted.update((p, self._adopt(p, saved.pop(i))) for i, p in zip(ids, params) if i in saved)
            return {**loaded, "state": saved}

        def after(_opt) -> None:  # before the other hooks
            self.state.update(adopted)
            self._plan = None

        hooks = (self.register_load_state_dict_pre_hook(before),
                 self.register_load_state_dict_post_hook(after, prepend=True))
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    @torch.no_grad()
    def _adopt(self, p: Tensor, saved: dict) -> dict:
        layout = self._layout(p)
        second = "exp_avg_sq_root" if "exp_avg_sq_root" in saved else "exp_avg_sq"
        scales = ("exp_avg_scale", "exp_avg_sq_root_scale") if second == "exp_avg_sq_root" else ()
        missing = [k for k in ("step", "exp_avg", second, *scales) if k not in saved]
        if missing:
            raise ValueError(f"the saved state of a parameter of shape {tuple(p.shape)} has no {missing}")
        step = saved["step"]
        if isinstance(step, Tensor):
            step = step.reshape(-1)[0].item() if step.numel() else 0
        entry = {"step": torch.full(layout["step"][1], int(step), dtype=torch.int32, device=p.device)}
        own = {k: v.to(p.device) for k, v in saved.items() if isinstance(v, Tensor) and k != "step"}
        same = all(k in own and own[k].dtype == d for k, (d, _) in layout.items() if k not in ("step", "master"))
        if same:
            entry.update({k: own[k].clone(memory_format=torch.contiguous_format) for k in layout if k not in ("step", "master")})
        else:
            if "exp_avg_sq_root" in own:
                m = _decode(own["exp_avg"], own["exp_avg_scale"])
                root = _decode(own["exp_avg_sq_root"], own["exp_avg_sq_root_scale"])
                v = root.square()
            else:
                m, v = own["exp_avg"].float(), own["exp_avg_sq"].float()
                root = v.sqrt()
            if "exp_avg_sq_root" in layout:
                entry["exp_avg"], entry["exp_avg_scale"] = _encode(m, False)
                entry["exp_avg_sq_root"], entry["exp_avg_sq_root_scale"] = _encode(root, True)
            else:
                entry["exp_avg"], entry["exp_avg_sq"] = (t.clone(memory_format=torch.contiguous_format) for t in (m, v))
        if "master" in layout:
            kept = own.get("master", p.detach())
            entry["master"] = kept.to(torch.float32, copy=True, memory_format=torch.contiguous_format)
        return entry

    # -- the step -------------------------------------------------------------------------

    def _step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        # A model has hundreds of parameters, and a step takes the GPU no longer than looking at each of them
        # takes Python: they are looked at natively, in lists.
        glue = _native.glue()
        if glue is None:
            raise RuntimeError(f"hip AdamW not supported: native library unavailable: {_native.glue_error()}")
        params = [p for group in self.param_groups for p in group["params"]]
        lie = glue.gradients(params)
        keep = None  # copies of strided gradients live until the launches are queued
        if lie is None:
            keep = [None if p.grad is None else _dense(p) for p in params]
            lie = np.array([0 if g is None else g.data_ptr() for g in keep], dtype=np.int64).tobytes()
        plan = self._plan
        if plan is None or not plan.current(self, glue, params, lie):
            plan = self._plan = _Plan(self, glue, params, lie)
        if not plan.kinds:  # the norm of no gradients
            device = params[0].device if params else None
            self.grad_norm = None if self.max_grad_norm is None else torch.zeros((), dtype=torch.float32, device=device)
            return loss
        plan.set_gradients(lie)
        device = plan.device
        hyper = plan.hyper(*[_hyper(g, device) for g in self.param_groups])
        if device.index != torch._C._cuda_getDevice():
            with torch.cuda.device(device):
                self._launch(plan, hyper, device)
        else:
            self._launch(plan, hyper, device)
        del keep
        # The kernels write past autograd's notice: what goes by a parameter's version has to see the change.
        torch.autograd.graph.increment_version(plan.active)
        return loss

    if _SHORTCUT:
        _heard_step = torch.optim.Optimizer.profile_hook_step(_step)

        def step(self, closure=None):
            # The base class's wrapper (a profiler's record, hooks) costs more than looking at the tensors does:
            # only where something listens.
            if (self._optimizer_step_pre_hooks or self._optimizer_step_post_hooks or _base._global_optimizer_pre_hooks
                    or _base._global_optimizer_post_hooks or torch.autograd.profiler._is_profiler_enabled):
                return self._heard_step(closure)
            return self._step(closure)

        step.hooked = True  # the base class leaves it as it is
    else:
        def step(self, closure=None):
            return self._step(closure)

    def _launch(self, plan: _Plan, hyper, device: torch.device) -> None:
        lib, stream = _native.lib(), _stream_ptr(device)
        partials, total, norm_ptr, at = None, 0, None, None
        self.grad_norm = None
        if self.max_grad_norm is not None:
            total = sum(partials for *_, partials in plan.norms)
            partials = torch.empty(total, dtype=torch.float64, device=device)
            self.grad_norm = torch.empty((), dtype=torch.float32, device=device)
            at = first = partials.data_ptr()
            norm_ptr = self.grad_norm.data_ptr()
            for pointer, count, code, n in plan.norms:
                _native.check(lib.ow_grad_norm(pointer, count, code, first, n, stream), "ow_grad_norm")
                first += 8 * n
        for kind in plan.kinds:
            _native.check(lib.ow_adamw_step(kind.pointer, kind.count, hyper, len(hyper), kind.code, kind.bits, kind.master, at,
                                            total, self.max_grad_norm or 0.0, norm_ptr, stream), "ow_adamw_step")
            norm_ptr = None


def _check_parameter(p: Tensor) -> None:
    if p.dtype not in SUPPORTED_DTYPES:
        raise ValueError(f"unsupported parameter dtype {p.dtype}; expected float32, bfloat16 or float16")
    if p.layout != torch.strided or not p.is_contiguous():
        raise ValueError(f"a parameter of shape {tuple(p.shape)} is not contiguous")


def _dense(p: Tensor) -> Tensor:
    """The gradient of ``p``, contiguous."""
    g = p.grad
    if g.layout != torch.strided:
        raise RuntimeError("AdamW takes dense gradients")
    if g.shape != p.shape or g.dtype != p.dtype or g.device != p.device:
        raise ValueError(f"the gradient of a {p.dtype} parameter of shape {tuple(p.shape)} is {g.dtype} {tuple(g.shape)} "
                         f"on {g.device}")
    return g.resolve_neg().contiguous()


def _without(lie: bytes) -> bytes:
    """Which of the gradients there are none of."""
    return (np.frombuffer(lie, dtype=np.int64) == 0).tobytes()


class _Plan:
    """What the steps of the same parameters share: their lists for the native calls.  It is made anew, with
    all its checks, where a parameter, a state or the set of parameters with gradients is another than it was:
    another tensor, at another address, or of another type, size or order at the same one."""

    def __init__(self, opt: AdamW, glue, params: list[Tensor], lie: bytes) -> None:
        self.params, self.device = params, None
        self.without, self.lie = _without(lie), None
        self.sizes = [len(group["params"]) for group in opt.param_groups]
        self.options = (opt.state_bits, opt.master_weights)
        self.hyper = _native.OwAdamwGroup * len(self.sizes)
        owner = [i for i, size in enumerate(self.sizes) for _ in range(size)]
        active = [i for i, p in enumerate(params) if not self.without[i] and p.numel()]
        kinds: dict[tuple, _Kind] = {}
        if active:
            self.device, reason = params[active[0]].device, gpu_reason(params[active[0]])
            if reason is not None:
                raise RuntimeError(f"hip AdamW not supported: {reason}")
        for i in active:
            p = params[i]
            if p.device != self.device:
                raise ValueError(f"parameters on {self.device} and {p.device}: an optimizer's parameters are on one GPU")
            if not p.is_contiguous():
                raise ValueError(f"a parameter of shape {tuple(p.shape)} is not contiguous")
            if not opt.state[p]:
                opt._first_state(p)
            layout = opt._layout(p)
            opt._check_state(p, layout)
            key = (p.dtype, 8 if "exp_avg_sq_root" in layout else 32, "master" in layout)
            if key not in kinds:
                _check_parameter(p)
                kinds[key] = _Kind(*key)
            kinds[key].add(i, p, opt.state[p], owner[i])
        self.active = [params[i] for i in active]
        _refuse_overlap(glue, self.active, [opt.state[p] for p in self.active])
        # One list, kinds of a dtype next to each other: their gradients' norm is one call.
        self.kinds = sorted(kinds.values(), key=lambda kind: kind.code)
        self.table = np.array([row for kind in self.kinds for row in kind.rows], dtype=np.int64)
        self.at = [i for kind in self.kinds for i in kind.at]
        self.norms: list[tuple[int, int, int, int]] = []  # address, tensors, dtype, partial sums
        first = 0
        for code, same in groupby(self.kinds, key=lambda kind: kind.code):
            start = first
            for kind in same:
                kind.pointer, kind.count = self.table[first:].ctypes.data, len(kind.rows)
                first += kind.count
            pointer, count = self.table[start:].ctypes.data, first - start
            self.norms.append((pointer, count, code, _native.lib().ow_grad_norm_partials(pointer, count)))
        self.layouts = glue.layouts(params)
        self.entries = list(opt.state.values())
        self.states = glue.state_layouts(self.entries)

    def current(self, opt: AdamW, glue, params: list[Tensor], lie: bytes) -> bool:
        """Whether everything but the gradients still lies where the plan has it."""
        entries = list(opt.state.values())
        return (len(params) == len(self.params) and all(map(is_, params, self.params))
                and (lie == self.lie or _without(lie) == self.without)
                and [len(group["params"]) for group in opt.param_groups] == self.sizes
                and (opt.state_bits, opt.master_weights) == self.options
                and len(entries) == len(self.entries) and all(map(is_, entries, self.entries))
                and glue.layouts(params) == self.layouts and glue.state_layouts(entries) == self.states)

    def set_gradients(self, lie: bytes) -> None:
        """Writes the gradients' addresses into the lists."""
        if lie != self.lie:
            where = np.frombuffer(lie, dtype=np.int64)
            self.table[:, _GRAD] = where[self.at]
            self.lie = lie


class _Kind:
    """Tensors of one dtype and state layout: one list for the native calls."""

    def __init__(self, dtype: torch.dtype, bits: int, master: bool) -> None:
        self.code, self.bits, self.master = _DTYPE_CODE[dtype], bits, master
        self.at: list[int] = []  # places among the parameters
        self.rows: list[list[int]] = []

    def add(self, i: int, p: Tensor, entry: dict[str, Tensor], group: int) -> None:
        second = ("exp_avg_sq_root", "exp_avg_scale", "exp_avg_sq_root_scale") if self.bits == 8 else ("exp_avg_sq",)
        ptr = [entry[k].data_ptr() for k in ("exp_avg", *second)] + [0] * (3 - len(second))
        self.at.append(i)
        self.rows.append([p.data_ptr(), 0, *ptr, entry["master"].data_ptr() if self.master else 0, entry["step"].data_ptr(),
                          p.numel(), group])


def _refuse_overlap(glue, params: list[Tensor], entries: list[dict]) -> None:
    """Tensors that share memory would be updated by two workgroups at once."""
    lie = memoryview(glue.addresses(params)).cast("q")
    spans = sorted((at, p.numel() * p.element_size(), i) for i, (at, p) in enumerate(zip(lie, params)))
    for (at, size, i), (other, _, j) in zip(spans, spans[1:]):
        if at + size > other:
            raise ValueError(f"parameters of shapes {tuple(params[i].shape)} and {tuple(params[j].shape)} share memory")
    states = [at for at in memoryview(glue.state_addresses(entries)).cast("q") if at]
    if len(set(states)) != len(states):
        raise ValueError("states of parameters share memory")


def _refuse_other_updates(group: dict) -> None:
    for name, plain in _PLAIN_UPDATE.items():
        if bool(group.get(name, plain)) != plain:
            raise ValueError(f"{name}={group[name]!r} is not supported")


def _hyper(group: dict, device: torch.device | None = None) -> tuple:
    """A group's hyperparameters as OwAdamwGroup's fields."""
    _refuse_other_updates(group)
    lr, (beta1, beta2), eps, decay = group["lr"], group["betas"], group["eps"], group["weight_decay"]
    lr_device = None
    if isinstance(lr, Tensor):
        if lr.numel() != 1 or not lr.is_floating_point():
            raise ValueError("lr must be a number or a floating point tensor of one value")
        if lr.is_cuda:
            if lr.dtype != torch.float32 or (device is not None and lr.device != device):
                raise ValueError(f"lr on a GPU must be float32 on the parameters' device, got {lr.dtype} on {lr.device}")
            lr_device, lr = lr.data_ptr(), 0.0
        else:
            lr = float(lr)
    if not (lr >= 0.0 and math.isfinite(lr)):
        raise ValueError(f"lr must be finite and not negative, got {lr}")
    if not (0.0 <= beta1 < 1.0 and 0.0 <= beta2 < 1.0):
        raise ValueError(f"betas must be in [0, 1), got {(beta1, beta2)}")
    if not (eps >= 0.0 and math.isfinite(eps)):
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    if not (decay >= 0.0 and math.isfinite(decay)):
        raise ValueError(f"weight_decay must be finite and not negative, got {decay}")
    return lr, beta1, beta2, eps, decay, lr_device
