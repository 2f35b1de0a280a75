"""Rotary positions without a GPU: frequencies, and what the entry point refuses before any device work."""
import ctypes as C
import math

import numpy as np
import pytest

import turboquant_plus_amd as tqa
from turboquant_plus_amd import _lib as L


def test_frequencies():
    f, mag = tqa.rotary_frequencies(8, 10000.0)
    assert np.allclose(f, [1.0, 0.1, 0.01, 0.001], rtol=1e-14) and mag == 1.0
    assert np.allclose(tqa.rotary_frequencies(8, 10000.0, tqa.RotaryScaling("linear", 4.0))[0], f / 4, rtol=1e-14)
    g = tqa.rotary_frequencies(8, 10000.0, tqa.RotaryScaling("ntk", 4.0))[0]
    assert g[0] == 1.0 and math.isclose(g[-1], f[-1] / 4, rel_tol=1e-12)        # the fastest stays, the slowest is divided
    # by parts: pairs over 32 turns in 4096 tokens keep their speed, those under one turn have it divided
    s = tqa.RotaryScaling("yarn", 16.0, trained_tokens=4096)
    f, (g, mag) = tqa.rotary_frequencies(128)[0], tqa.rotary_frequencies(128, scaling=s)
    turns = f * 4096 / (2 * math.pi)
    assert np.array_equal(g[turns >= 40], f[turns >= 40]) and np.allclose(g[turns <= 0.9], f[turns <= 0.9] / 16, rtol=1e-14)
    assert (np.diff(g) < 0).all() and math.isclose(mag, 0.1 * math.log(16.0) + 1.0)
    assert tqa.rotary_frequencies(128, scaling=tqa.RotaryScaling("yarn", 16.0, trained_tokens=4096, magnitude=1.0))[1] == 1.0


@pytest.mark.parametrize("kw", [dict(kind="other", factor=2.0), dict(kind="linear", factor=0.0), dict(kind="linear", factor=float("nan")),
                                dict(kind="yarn", factor=2.0), dict(kind="yarn", factor=2.0, trained_tokens=4096, slow_turns=64.0)])
def test_scalings_that_make_no_sense(kw):
    with pytest.raises(ValueError):
        tqa.RotaryScaling(**kw)


@pytest.mark.parametrize("args", [(7,), (0,), (64, 1.0), (64, float("inf")), (2, 10000.0, tqa.RotaryScaling("ntk", 2.0))])
def test_frequencies_that_make_no_sense(args):
    with pytest.raises(ValueError):
        tqa.rotary_frequencies(*args)


def params(**kw):
    p = dict(tokens=4, n_q_heads=2, n_k_heads=1, head_dim=128, rotary_dim=64, dtype=L.TQ_F16, magnitude=1.0)
    return L.TQRotaryParams(**{**p, **kw})


@pytest.mark.parametrize("kw,code,text", [
    (dict(tokens=-1), L.ERR_ARG, "negative"), (dict(n_q_heads=-1), L.ERR_ARG, "negative"), (dict(head_dim=0), L.ERR_ARG, "head_dim"),
    (dict(rotary_dim=63), L.ERR_ARG, "even"), (dict(rotary_dim=0), L.ERR_ARG, "even"), (dict(rotary_dim=130), L.ERR_ARG, "even"),
    (dict(rotary_dim=2048, head_dim=2048), L.ERR_UNSUPPORTED, "1024"), (dict(dtype=L.TQ_F64), L.ERR_ARG, "dtype"),
    (dict(n_q_heads=70000), L.ERR_UNSUPPORTED, "heads")])
def test_entry_point_refuses(kw, code, text):
    x = C.c_void_p(4096)
    assert L.lib().tq_rotary(C.byref(params(**kw)), x, x, x, x, x, x, None) == code
    assert text in L.last_error()


def test_entry_point_refuses_pointers():
    x, odd, call = C.c_void_p(4096), C.c_void_p(4097), L.lib().tq_rotary
    assert call(None, x, x, x, x, x, x, None) == L.ERR_ARG
    assert call(C.byref(params()), x, None, x, x, x, x, None) == L.ERR_ARG
    assert call(C.byref(params()), x, x, x, x, None, x, None) == L.ERR_ARG
    assert call(C.byref(params()), odd, x, x, x, x, x, None) == L.ERR_ALIGN
    assert call(C.byref(params()), x, x, x, x, odd, x, None) == L.ERR_ALIGN
    assert call(C.byref(params(tokens=0)), None, None, None, None, None, None, None) == 0
    assert call(C.byref(params(n_q_heads=0, n_k_heads=0)), None, None, None, None, None, None, None) == 0
