"""AdamW: what the optimizer refuses, its state dictionaries and 8-bit format, on the CPU, and the C
entry points' argument checks."""

from __future__ import annotations

import copy
import ctypes
import io

import numpy as np
import pytest
import torch

from omniwave_amd import AdamW, _native
from omniwave_amd.optim import _decode, _encode


def param(*shape, dtype=torch.float32):
    return torch.nn.Parameter(torch.randn(shape).to(dtype))


@pytest.mark.parametrize("kwargs,text", [
    (dict(lr=-1.0), "lr"), (dict(lr=float("inf")), "lr"), (dict(lr=torch.ones(2)), "lr"),
    (dict(betas=(1.0, 0.9)), "betas"), (dict(betas=(0.9, -0.1)), "betas"), (dict(eps=-1e-8), "eps"),
    (dict(weight_decay=-1.0), "weight_decay"), (dict(state_bits=4), "state_bits"),
    (dict(max_grad_norm=0.0), "max_grad_norm"), (dict(max_grad_norm=float("inf")), "max_grad_norm"),
])
def test_refused_hyperparameters(kwargs, text) -> None:
    with pytest.raises(ValueError, match=text):
        AdamW([param(3)], **kwargs)


def test_refused_parameters() -> None:
    with pytest.raises(ValueError, match="dtype"):
        AdamW([param(3, dtype=torch.float64)])
    with pytest.raises(ValueError, match="not contiguous"):
        AdamW([torch.nn.Parameter(torch.randn(4, 6).t())])
    p = param(3)
    with pytest.raises(ValueError, match="twice"):
        with pytest.warns(UserWarning):
            AdamW([p, p])
    opt = AdamW([p])
    with pytest.raises(ValueError, match="not contiguous"):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.randn(4, 6).t())]})
    assert len(opt.param_groups) == 1


def test_the_cpu_has_no_kernel() -> None:
    p = param(5)
    opt = AdamW([p])
    assert opt.step() is None  # nothing has a gradient
    p.grad = torch.ones(5)
    with pytest.raises(RuntimeError, match="not supported"):
        opt.step()


def test_8_bit_format() -> None:
    torch.manual_seed(0)
    values = torch.randn(5, 300) * torch.logspace(-6, 3, 5)[:, None]
    values[0, :7] = 0
    codes, scale = _encode(values, False)
    assert codes.dtype == torch.float8_e4m3fn and scale.shape == (6,)
    held = _decode(codes, scale)
    flat = values.reshape(-1)
    most = torch.nn.functional.pad(flat.abs(), (0, 36)).reshape(6, 256).amax(1)
    assert torch.allclose(scale, most / 448, rtol=1e-6)
    step = torch.maximum(flat.abs() * 2 ** -4, scale.repeat_interleave(256)[:1500] * 2 ** -10)
    assert ((held.reshape(-1) - flat).abs() <= step * (1 + 1e-5)).all()
    root, rscale = _encode(values.abs(), True)
    assert ((root.float() > 0) == (values != 0)).all()
    zeros, zscale = _encode(torch.zeros(256), True)
    assert not zeros.float().any() and not zscale.any() and not _decode(zeros, zscale).any()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_states_of_torch_are_taken_over(bits, dtype) -> None:
    params = [param(70, 70, dtype=dtype), param(33, dtype=dtype)]
    other = torch.optim.AdamW(params, lr=0.01)
    for _ in range(3):
        for p in params:
            p.grad = torch.randn_like(p)
        other.step()
    opt = AdamW(params, state_bits=bits, master_weights=True)
    opt.load_state_dict(other.state_dict())
    assert opt.param_groups[0]["lr"] == 0.01
    for p in params:
        entry, theirs = opt.state[p], other.state[p]
        opt._check_state(p)
        assert (entry["step"] == 3).all()
        if bits == 8 and p.numel() >= 4096:
            assert entry["exp_avg"].dtype == torch.float8_e4m3fn
            m = _decode(entry["exp_avg"], entry["exp_avg_scale"])
            root = _decode(entry["exp_avg_sq_root"], entry["exp_avg_sq_root_scale"])
            # half a step of e4m3fn, relative, or half its least step of the block's largest value
            assert ((m - theirs["exp_avg"].float()).abs() <= (m.abs() * 2 ** -4).clamp(min=m.abs().max() / 448 * 2 ** -9)).all()
            assert ((root.square() - theirs["exp_avg_sq"].float()).abs() <= theirs["exp_avg_sq"].float() * 0.14 + 1e-9).all()
        else:
            assert torch.equal(entry["exp_avg"], theirs["exp_avg"].float())
            assert torch.equal(entry["exp_avg_sq"], theirs["exp_avg_sq"].float())
        assert ("master" in entry) == (dtype != torch.float32)


def test_state_dict_round_trip_keeps_dtypes() -> None:
    params = [param(70, 70, dtype=torch.bfloat16), param(33, dtype=torch.bfloat16)]
    opt = AdamW(params, state_bits=8, master_weights=True)
    for p in params:
        opt.state[p] = opt._adopt(p, dict(step=7, exp_avg=torch.randn(p.shape), exp_avg_sq=torch.rand(p.shape)))
    again = AdamW(params, state_bits=8, master_weights=True)
    again.load_state_dict(copy.deepcopy(opt.state_dict()))
    for p in params:
        assert opt.state[p].keys() == again.state[p].keys()
        for k, t in opt.state[p].items():
            assert again.state[p][k].dtype == t.dtype and torch.equal(again.state[p][k].float(), t.float()), k
    back = AdamW(params)  # 8 bits to 32
    back.load_state_dict(opt.state_dict())
    e = opt.state[params[0]]
    assert torch.equal(back.state[params[0]]["exp_avg"], _decode(e["exp_avg"], e["exp_avg_scale"]))
    held = io.BytesIO()
    torch.save(opt.state_dict(), held)
    held.seek(0)
    again.load_state_dict(torch.load(held, weights_only=True))
    assert torch.equal(again.state[params[0]]["exp_avg"].float(), e["exp_avg"].float())
    kept = copy.deepcopy(opt)
    assert (kept.state_bits, kept.master_weights, kept.max_grad_norm) == (8, True, None)


def test_damaged_states_are_refused() -> None:
    p = param(70, 70)
    opt = AdamW([p])
    good = opt._adopt(p, dict(step=1, exp_avg=torch.zeros(70, 70), exp_avg_sq=torch.zeros(70, 70)))
    opt.state[p] = good
    opt._check_state(p)
    for name, bad in (("exp_avg", torch.zeros(70)), ("exp_avg_sq", torch.zeros(70, 70).bfloat16()),
                      ("step", torch.zeros(1, dtype=torch.int32)), ("exp_avg", torch.zeros(70, 70).t()), ("exp_avg_sq", None)):
        opt.state[p] = {**good, name: bad}
        with pytest.raises(ValueError, match=name):
            opt._check_state(p)
    with pytest.raises(ValueError, match="has no"):
        opt._adopt(p, dict(step=1))


def test_c_entry_points_check_their_arguments() -> None:
    lib = _native.lib()
    assert ctypes.sizeof(_native.OwAdamwTensor) == 80 and ctypes.sizeof(_native.OwAdamwGroup) == 48
    f32, bf16 = _native.OW_DTYPE_F32, _native.OW_DTYPE_BF16
    good = [256, 256, 256, 256, 256, 256, 256, 256, 100, 0]

    def table(**kw):
        row = dict(zip([n for n, _ in _native.OwAdamwTensor._fields_], good))
        row.update(kw)
        t = np.array([list(row.values())], dtype=np.int64)
        table.keep = t
        return t.ctypes.data

    def step(t, dtype=f32, bits=32, master=0, hyper=(1e-3, 0.9, 0.999, 1e-8, 0.0), groups=1, partials=None, n=0, most=0.0):
        h = (_native.OwAdamwGroup * 1)(hyper)
        return lib.ow_adamw_step(t, 1, h, groups, dtype, bits, master, partials, n, most, None, None)

    def refused(rc, text, code=1):
        assert rc == code and text in lib.ow_last_error(), lib.ow_last_error()

    refused(step(table(), dtype=9), b"dtype", 2)
    refused(step(table(), bits=4), b"bits", 2)
    refused(step(table(), master=1), b"master", 2)
    refused(step(table(master=0), dtype=bf16, master=1), b"master")
    refused(step(table(numel=0)), b"0 values")
    refused(step(table(numel=(1 << 40) + 1)), b"2^40", 2)
    refused(step(table(grad=0)), b"gradient")
    refused(step(table(step=0)), b"NULL")
    refused(step(table(exp_avg_scale=0), bits=8), b"scales")
    refused(step(table(group=1)), b"group 1 of 1")
    refused(step(table(), hyper=(1e-3, 1.0, 0.999, 1e-8, 0.0)), b"beta1")
    refused(step(table(), partials=256, n=0, most=1.0), b"clipping")
    refused(step(table(), partials=256, n=8, most=0.0), b"clipping")
    assert lib.ow_adamw_step(None, 0, None, 0, f32, 32, 0, None, 0, 0.0, None, None) == 0
    assert lib.ow_grad_norm_partials(None, 3) == 0 and lib.ow_grad_norm_partials(table(), 1) == 1024
    many = np.array([good] * 600, dtype=np.int64)
    assert lib.ow_grad_norm_partials(many.ctypes.data, 600) == 3 * 1024
    refused(lib.ow_grad_norm(table(), 1, f32, ctypes.c_void_p(256), 1000, None), b"1024 are needed")
    refused(lib.ow_grad_norm(table(), -1, f32, None, 0, None), b"negative")
