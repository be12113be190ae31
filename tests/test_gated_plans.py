"""Which kernels of the gated feed-forward product a size takes: the cases that ``test_gpu_gated_plans.py`` runs reach every tile,
whole, cut and both, in every product.  A change of the rules that moves a case to another kernel is seen here.

A plan is, for forward, gates, dx and the weights' gradients: the tile (L 256 x 256, M 128 x 128, S 64 x 128; "few": the
kernel for few tokens), and whether its tiles take their whole k, are cut into parts of it, or both; "kept": no product is
formed again.  Without a GPU the library plans for 256 compute units, as an MI355X has.
"""

from __future__ import annotations

import ctypes

import pytest

from omniwave_amd import _native

# rows, channels, hidden; the plans of 16-bit types, of fp32
CASES = [
    (9001, 200, 700, "L whole, L whole, S whole, S cut", "L whole, kept, L cut, M cut"),
    (9000, 199, 701, "L whole, L whole, S whole, S cut", "L whole, kept, L cut, M cut"),
    (200, 1536, 2816, "S whole, kept, S cut, L whole", "M cut, kept, M cut, M both"),
    (201, 1537, 2815, "S whole, kept, S cut, L whole", "M cut, kept, M cut, L whole"),
    (33000, 64, 64, "M whole, M whole, M whole, L cut", "M whole, M whole, M whole, S cut"),
    (33001, 63, 65, "S whole, S whole, M whole, S cut", "S whole, S whole, M whole, S cut"),
    (33000, 200, 64, "M whole, M whole, L whole, S cut", "S both, kept, L whole, S cut"),
    (12000, 200, 2816, "M whole, M whole, L cut, M cut", "L both, kept, L cut, L cut"),
    (12001, 201, 2817, "M whole, M whole, L cut, M cut", "L both, kept, L cut, L cut"),
    (12000, 2816, 256, "M whole, kept, L both, M cut", "L cut, kept, L both, L cut"),
    (12001, 2815, 255, "M whole, kept, L both, M cut", "L cut, kept, L both, L cut"),
    (33000, 1024, 512, "L both, M whole, L both, L cut", "L both, kept, L both, L cut"),
    (33001, 1023, 511, "L both, M whole, L both, L cut", "L both, kept, L both, L cut"),
    (3000, 1536, 2816, "L both, kept, L cut, M both", "L both, kept, L cut, M both"),
    (3001, 1537, 2815, "L both, kept, L cut, M both", "L both, kept, L cut, L cut"),
    (3000, 1536, 1536, "L whole, kept, S both, S both", "M both, kept, L cut, L cut"),
    (1500, 1536, 2816, "M both, kept, M cut, M both", "M both, kept, L cut, M both"),
    (1501, 1535, 2817, "M both, L whole, M cut, L whole", "M both, kept, L cut, M both"),
    (6272, 5000, 130, "M cut, kept, L whole, S cut", "M cut, kept, L whole, L cut"),
    (1000, 1536, 6000, "L whole, kept, M cut, L both", "M both, kept, L cut, L both"),
    (12000, 1536, 130, "M whole, kept, M whole, S cut", "S both, kept, L both, L cut"),
    (33000, 1536, 64, "S both, kept, M whole, S cut", "S both, kept, L both, S cut"),
    (12000, 1024, 700, "M both, M whole, L whole, M cut", "L both, kept, L whole, L cut"),
    (33000, 64, 1024, "M whole, M whole, S both, S cut", "M whole, M whole, S both, M cut"),
    (33000, 200, 700, "M whole, M whole, M both, M cut", "L both, kept, M both, L cut"),
    (4000, 64, 6000, "M whole, M whole, S cut, M cut", "L whole, L whole, M cut, M cut"),
    (12000, 64, 2048, "M whole, M whole, M cut, S cut", "L whole, L whole, M cut, M cut"),
    (2000, 2048, 520, "S whole, kept, S whole, S whole", "M cut, kept, L cut, M cut"),
    (200, 5000, 1024, "S cut, kept, S cut, L whole", "S cut, kept, M cut, L whole"),
]
CODES = {"f32": 0, "bf16": 1, "f16": 2}
TILES = {(0, 0): "few", (256, 256): "L", (128, 128): "M", (64, 128): "S"}


def descriptor(rows, c, hidden, dtype):
    # Addresses that no call looks at, aligned as allocations are.
    return _native.OwGatedLinear(rows, c, 1 << 20, 1 << 20, 1 << 20, c, hidden, CODES[dtype])


def plans(rows, c, hidden, dtype):
    """A plan for each product."""
    d, got = descriptor(rows, c, hidden, dtype), []
    for product, code in _native.OW_GATED.items():
        if product == "gates" and _native.lib().ow_gated_linear_kept(ctypes.byref(d)):
            got.append("kept")
            continue
        p = _native.OwGatedPlan()
        assert _native.lib().ow_gated_linear_plan(ctypes.byref(d), code, ctypes.byref(p)) == 0
        name = TILES[p.tile_rows, p.tile_cols]
        if name != "few":
            assert p.whole + p.cut > 0 and (p.parts > 1) == (p.cut > 0)
            name += " whole" if not p.cut else " both" if p.whole else " cut"
        got.append(name)
    return got


@pytest.mark.parametrize("rows,c,hidden,narrow,wide", CASES)
def test_plans(rows, c, hidden, narrow, wide) -> None:
    for dtype in CODES:
        assert ", ".join(plans(rows, c, hidden, dtype)) == (wide if dtype == "f32" else narrow)


def test_the_cases_reach_every_kernel() -> None:
    seen = {True: set(), False: set()}
    for _, _, _, narrow, wide in CASES:
        for of, plan in ((False, narrow), (True, wide)):
            forward, gates, dx, dw = plan.split(", ")
            seen[of] |= {("keep" if gates == "kept" else "forward", forward), ("gates", gates), ("dx", dx), ("dw", dw)}
    for of in (False, True):
        assert {("gates", f"{tile} whole") for tile in "LMS"} <= seen[of]  # gates are never cut
        assert {("forward", f"{tile} whole") for tile in "LMS"} <= seen[of]
        assert {("dx", "L both"), ("dx", "L cut"), ("dx", "L whole"), ("dx", "M both"), ("dx", "M cut"), ("dx", "M whole"),
                ("dx", "S both"), ("dw", "L both"), ("dw", "L cut"), ("dw", "L whole"), ("dw", "M both"), ("dw", "M cut"),
                ("dw", "S cut"), ("keep", "L both"), ("keep", "L whole"), ("keep", "M both"), ("keep", "M cut"), ("keep", "S both"),
                ("keep", "S cut")} <= seen[of]
    # Products of channels below the width from which both are kept are cut in 16 bits alone: fp32 keeps them from 128 on.
    assert {("forward", "L both"), ("forward", "M both"), ("keep", "M whole"), ("keep", "S whole"), ("dx", "S cut"),
            ("dx", "S whole"), ("dw", "S both"), ("dw", "S whole")} <= seen[False]
    assert ("keep", "L cut") in seen[True]


def test_refusals() -> None:
    lib, p = _native.lib(), _native.OwGatedPlan()
    d = descriptor(70, 64, 64, "bf16")
    assert lib.ow_gated_linear_plan(ctypes.byref(d), 0, ctypes.byref(p)) == 0
    for desc, product, plan in ((None, 0, p), (d, 4, p), (d, -1, p), (d, 0, None), (descriptor(0, 64, 64, "bf16"), 0, p),
                                (descriptor(70, 0, 64, "bf16"), 0, p), (descriptor(70, 64, 0, "bf16"), 0, p)):
        refs = [None if s is None else ctypes.byref(s) for s in (desc, plan)]
        assert lib.ow_gated_linear_plan(refs[0], product, refs[1]) != 0
