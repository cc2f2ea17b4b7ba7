"""Rotary positions on the host: frequencies and refusals (no GPU call)."""
import ctypes as C
import math

import numpy as np
import pytest

from eos_amd import _lib
from eos_amd._lib import EosHipError
from eos_amd.rotary import Rotary, frequencies


def test_frequencies_are_the_textbooks():
    f, c = frequencies(64)
    np.testing.assert_allclose(f, [10000.0 ** (-2 * i / 64) for i in range(32)], rtol=1e-15)
    assert c == 1.0
    g, _ = frequencies(64, scaling="linear", stretch=4)
    np.testing.assert_allclose(g, f / 4, rtol=1e-15)
    g, _ = frequencies(64, scaling="base", stretch=8)
    assert g[0] == 1.0
    np.testing.assert_allclose(g[-1], f[-1] / 8, rtol=1e-12)
    assert (np.diff(g) < 0).all()
    assert frequencies(2, scaling="base", stretch=8)[0] == [1.0]


@pytest.mark.parametrize("scaling", ["ramp", "wavelength"])
def test_frequencies_by_their_turns(scaling):
    original, stretch = 4096, 16.0
    f, _ = frequencies(128, 500000.0)
    g, c = frequencies(128, 500000.0, scaling, stretch, original, low=1, high=32)
    turns = original * f / (2 * math.pi)
    part = f / g  # 1: as it is, 16: divided
    # (the ramp runs over whole indices: a border's neighbours may still move)
    fast, slow = turns > 40, turns < 0.8
    np.testing.assert_allclose(part[fast], 1.0, rtol=1e-12)
    np.testing.assert_allclose(part[slow], stretch, rtol=1e-12)
    assert fast.any() and slow.any() and (np.diff(part) >= -1e-9).all()
    assert c == (1.0 if scaling == "wavelength" else 0.1 * math.log(stretch) + 1)


@pytest.mark.parametrize("kw", [dict(rotary_dim=0), dict(rotary_dim=7), dict(rotary_dim=8, base=1.0),
                                dict(rotary_dim=8, stretch=0.5), dict(rotary_dim=8, scaling="other"),
                                dict(rotary_dim=8, scaling="ramp"),
                                dict(rotary_dim=8, scaling="ramp", original=9, low=2, high=2)])
def test_frequencies_refused(kw):
    with pytest.raises(ValueError):
        frequencies(**kw)


@pytest.mark.parametrize("kw,what", [
    (dict(head_dim=4), "head_dim"), (dict(head_dim=100), "head_dim"), (dict(head_dim=1032), "head_dim"),
    (dict(rotary_dim=0), "rotary_dim"), (dict(rotary_dim=7), "rotary_dim"),
    (dict(rotary_dim=66), "rotary_dim"), (dict(layout=2), "layout"),
    (dict(factor=float("inf")), "factor"), (dict(frequencies=None), "frequencies"),
    (dict(freq=[1.0, float("nan")]), r"frequencies\[1\]"), (dict(freq=[65.0, 1.0]), r"frequencies\[0\]"),
    (dict(), "NULL argument")])
def test_bind_refused(kw, what):
    f = np.array(kw.pop("freq", [1.0, 0.5] + [0.25] * 30), np.float64)
    a = dict(head_dim=64, rotary_dim=2 * len(f), layout=1, factor=1.0,
             frequencies=f.ctypes.data) | kw
    out = C.c_void_p(1)
    with pytest.raises(EosHipError, match=what):
        _lib.call("eoship_rotary_bind", None, C.byref(_lib.EosHipRotaryDesc(**a)), C.byref(out))
    assert not out


def test_null_and_names_refused():
    with pytest.raises(EosHipError, match="NULL"):
        _lib.call("eoship_rotary_device", None, None, None, 4096, 1, 0, 1, 4096, 64, 1, 4096, 64,
                  None, 0, 0, None, 0)
    _lib.call("eoship_rotary_release", None, None)
    with pytest.raises(ValueError, match="layout"):
        Rotary(None, 64, np.ones(32), "thirds")
    with pytest.raises(ValueError, match="freq"):
        Rotary(None, 64, np.ones((2, 16)))
