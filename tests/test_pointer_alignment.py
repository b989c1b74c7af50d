"""Pointers off the boundary of their type are refused by the C ABI's training calls, as a read through them would
fault on a device."""

import pytest

from test_operators_cpu import BF, F32, INV, _distill, _mod_bwd, _mod_fwd, _norm


@pytest.mark.parametrize("name", ["slopes", "seg", "prefix", "lse"])
@pytest.mark.parametrize("at", [17, 18])
def test_attention(name, at):
    assert _mod_fwd(**{name: at}) == INV and _mod_bwd(**{name: at}) == INV


@pytest.mark.parametrize("at", [17, 18])
def test_slopes_gradient(at):
    assert _mod_bwd(slopes=16, dslopes=at) == INV


@pytest.mark.parametrize("name", ["wq", "wk", "dwq", "dwk"])
def test_norm_weights(name):
    for fn in ("fwd", "bwd") if name in ("wq", "wk") else ("bwd",):
        assert _norm(fn, **{name: 17}) == INV
        assert _norm(fn, wdtype=F32, **{name: 18}) == INV


@pytest.mark.parametrize("fn,name,at", [("fwd", "teacher", 18), ("fwd", "w", 18), ("fwd", "rows", 17), ("fwd", "loss", 18),
                                        ("bwd", "grad", 18), ("fwd", "dz", 17), ("bwd", "dz", 17), ("fwd", "ids", 18),
                                        ("bwd", "ids", 18)])
def test_distillation(fn, name, at):
    assert _distill(fn, **{name: at}) == INV


@pytest.mark.parametrize("fn", ["fwd", "bwd"])
def test_distillation_of_wider_types(fn):
    assert _distill(fn, ids=20, i64=1) == INV and _distill(fn, dtype=F32, dz=18) == INV and _distill(fn, dtype=BF, z=17) == INV
