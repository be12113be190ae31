"""The native calls of the small operators (``_glue``) on the CPU: the module loads, and gives back to the
checked path whatever is not its plain case."""

from __future__ import annotations

import pytest
import torch

from omniwave_amd import _native


def test_the_module_loads() -> None:
    assert _native.glue_error() is None and _native.glue() is not None


def test_other_inputs_are_handed_back() -> None:
    glue, x, w = _native.glue(), torch.zeros(2, 3, 8), torch.ones(8)
    assert glue.norms(x, x, w, w, None, w, 1e-6) is None  # not on a GPU
    assert glue.norms(None, None, None, None, None, None, 1e-6) is None
    assert glue.norms(x, "delta", w, w, None, w, 1e-6) is None
    assert glue.norms(x, x, w, w, None, w, "eps") is None
    t = torch.zeros(2, 3, dtype=torch.int64)
    assert glue.cross_entropy(x, t, None, None, 1.0, 0.0, -100, 2) is None
    assert glue.cross_entropy(x, None, None, None, 1.0, 0.0, -100, 2) is None
    assert glue.cross_entropy(x, t, None, None, 1.0, 0.0, None, 2) is None
    with pytest.raises(TypeError):
        glue.norms(x)
    with pytest.raises(TypeError):
        glue.cross_entropy(x, t)


def test_addresses() -> None:
    glue = _native.glue()
    ts = [torch.zeros(3), torch.zeros(2, 2)[1:], torch.zeros(0)]
    want = b"".join(t.data_ptr().to_bytes(8, "little") for t in ts)
    assert glue.addresses(ts) == want
    assert glue.state_addresses([{"a": ts[0], "b": 3}, {}, {"c": ts[1]}]) == want[:8] + bytes(8) + want[8:16]
    for bad in (ts[0], [1], None):
        with pytest.raises(TypeError):
            glue.addresses(bad)
        with pytest.raises(TypeError):
            glue.state_addresses(bad)


def test_gradients() -> None:
    glue = _native.glue()
    p, q = torch.zeros(3, 4, requires_grad=True), torch.zeros(2, requires_grad=True)
    assert glue.gradients([p, q]) == bytes(16)
    p.grad = torch.ones(3, 4)
    assert glue.gradients([p, q]) == p.grad.data_ptr().to_bytes(8, "little") + bytes(8)
    p.grad = torch.ones(4, 3).t()
    assert glue.gradients([p, q]) is None
    p.grad = torch.eye(3, 4).to_sparse()
    assert glue.gradients([p, q]) is None
    p.grad = torch.ones(3, 4)
    p.grad.data = torch.ones(2)  # torch itself lets a gradient's data be swapped for another size
    assert glue.gradients([p, q]) is None
    with pytest.raises(TypeError):
        glue.gradients([1])
