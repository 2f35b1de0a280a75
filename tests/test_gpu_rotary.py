"""Rotary positions against the formula in 64 bits.

Tolerances: a result is a sum of two products in 32 bits of a value, a cosine or sine (each off by at most 2^-23, the magnitude's
product by another 2^-24) and one rounding to the type: |error| <= eps(type) / 2 |result| + 2^-21 (|u| + |w|) magnitude.
"""
import math

import numpy as np
import pytest

import turboquant_plus_amd as tqa
from turboquant_plus_amd import _lib as L

pytestmark = pytest.mark.gpu
tt = L.torch()
DTYPES = {"fp16": tt.float16, "bf16": tt.bfloat16, "fp32": tt.float32}
SCALINGS = {"none": None, "linear": tqa.RotaryScaling("linear", 4.0), "ntk": tqa.RotaryScaling("ntk", 4.0),
            "yarn": tqa.RotaryScaling("yarn", 16.0, trained_tokens=4096)}


def frequencies(r, base, s):
    """Radians per position, pair by pair, from the definitions."""
    if s is not None and s.kind == "ntk":
        base = base * s.factor ** (r / (r - 2))
    f = [base ** (-2 * i / r) for i in range(r // 2)]
    if s is None or s.kind == "ntk":
        return f, 1.0
    if s.kind == "linear":
        return [x / s.factor for x in f], 1.0
    pair = lambda turns: r * math.log(s.trained_tokens / (turns * 2 * math.pi)) / (2 * math.log(base))
    lo, hi = max(math.floor(pair(s.fast_turns)), 0), min(math.ceil(pair(s.slow_turns)), r - 1)
    w = [min(max((i - lo) / max(hi - lo, 1e-3), 0), 1) for i in range(r // 2)]
    return [x * (1 - a) + x / s.factor * a for x, a in zip(f, w)], 0.1 * math.log(s.factor) + 1


def turned(x, pos, r, interleaved, scaling, inverse, base=10000.0):
    f, mag = frequencies(r, base, scaling)
    a = np.outer(pos.astype(np.float64), f)[:, None]
    c, s = np.cos(a) * mag, np.sin(a) * mag * (-1 if inverse else 1)
    y, size = x.copy(), np.zeros_like(x)
    u, w = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    y[..., u], y[..., w] = x[..., u] * c - x[..., w] * s, x[..., w] * c + x[..., u] * s
    size[..., u] = size[..., w] = (np.abs(x[..., u]) + np.abs(x[..., w])) * mag
    return y, size


def check(got, x, pos, rot, inverse=False, scaling=None):
    want, size = turned(x.double().cpu().numpy(), pos.cpu().numpy(), rot.rotary_dim, rot.interleaved, scaling, inverse)
    err = np.abs(got.double().cpu().numpy() - want)
    bound = tt.finfo(x.dtype).eps / 2 * np.abs(want) + 2.0 ** -21 * size + 2.0 ** -25    # fp16's subnormals
    assert (err <= bound).all(), float((err - bound).max())
    assert got.dtype == x.dtype


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,hq,hkv,d,r", [(1, 32, 8, 128, 128), (7, 4, 1, 128, 64), (2049, 5, 5, 64, 64), (300, 3, 2, 256, 32),
                                               (5, 2, 1, 80, 20), (3, 1, 1, 6, 6), (4, 2, 2, 7, 2), (2, 1, 1, 2048, 1024)])
def test_against_the_formula(dtype, interleaved, tokens, hq, hkv, d, r):
    gen = tt.Generator("cuda").manual_seed(tokens)
    q, k = (tt.randn((tokens, h, d), generator=gen, device="cuda").to(DTYPES[dtype]) for h in (hq, hkv))
    pos = tt.randint(0, 100000, (tokens,), generator=gen, device="cuda")
    rot = tqa.Rotary(r, interleaved=interleaved)
    q2, k2 = rot(q, k, pos)
    check(q2, q, pos, rot)
    check(k2, k, pos, rot)
    assert tt.equal(q2[..., r:], q[..., r:]) and tt.equal(k2[..., r:], k[..., r:])


@pytest.mark.parametrize("scaling", SCALINGS)
@pytest.mark.parametrize("inverse", [False, True])
def test_scaled_frequencies_and_far_positions(scaling, inverse):
    pos = tt.tensor([0, 1, 4095, 65536, 999_999, 2 ** 31 - 1, -5, 2 ** 40 + 3], device="cuda")
    gen = tt.Generator("cuda").manual_seed(3)
    q = tt.randn((8, 3, 128), generator=gen, device="cuda")
    s = SCALINGS[scaling]
    rot = tqa.Rotary(128, scaling=s)
    got, none = rot(q, None, pos, inverse=inverse)
    assert none is None
    # 2^40 radians are known to 2^-13 only in the oracle's own 64 bits: that row is left to the one below
    check(got[:7], q[:7], pos[:7], rot, inverse, s)
    back, _ = rot(got[:7], None, pos[:7], inverse=not inverse)
    mag = rot.magnitude ** 2
    assert (back / mag - q[:7]).abs().max() < 2 ** -18      # two turns, magnitudes up to 5
    if scaling == "none":
        turn = (pos[7].item() * int(round(float(rot.turns[0]) * 2 ** 60)) % 2 ** 60) / 2 ** 60   # frequency 1, whole arithmetic
        a = 2 * math.pi * turn * (-1 if inverse else 1)
        want = q[7, 0, 0].item() * math.cos(a) - q[7, 0, 64].item() * math.sin(a)
        assert abs(got[7, 0, 0].item() - want) < 5e-4       # 2^40 turns / 2 pi in 53 bits leave 2^-13 of a turn


def test_int32_positions_strides_and_in_place():
    gen = tt.Generator("cuda").manual_seed(4)
    for dtype, extra in ((tt.float16, 8), (tt.bfloat16, 0), (tt.float32, 3)):      # 3: rows that no 16-byte load may take
        qkv = tt.randn((37, 6 * 128 + extra), generator=gen, device="cuda").to(dtype)
        q, k = qkv[:, :512].unflatten(1, (4, 128)), qkv[:, 512:640].unflatten(1, (1, 128))
        pos = tt.randint(0, 5000, (74,), generator=gen, device="cuda").int()[::2]
        rot = tqa.Rotary(64)
        want = [x.clone() for x in rot(q.contiguous(), k.contiguous(), pos.contiguous())]
        before = qkv.clone()
        got = rot(q, k, pos)
        assert all(tt.equal(a, b) for a, b in zip(got, want)) and tt.equal(qkv, before)
        rot(q, k, pos, out=(q, k))
        assert tt.equal(q, want[0]) and tt.equal(k, want[1]) and tt.equal(qkv[:, 640:], before[:, 640:])
        # heads before tokens
        qt = want[0].transpose(0, 1).contiguous().transpose(0, 1)
        assert tt.equal(rot(qt, None, pos, inverse=True)[0], rot(want[0], None, pos, inverse=True)[0])


def test_gradient_is_the_inverse_turn():
    """sum(g . R x) has the gradient R^T g, against differences of the formula in 64 bits."""
    rng = np.random.default_rng(5)
    x, g, pos = rng.standard_normal((3, 2, 16)), rng.standard_normal((3, 2, 16)), np.array([1, 700, 123456])
    for interleaved in (False, True):
        rot = tqa.Rotary(12, interleaved=interleaved)
        got = rot(tt.tensor(g, dtype=tt.float32, device="cuda"), None, tt.tensor(pos, device="cuda"), inverse=True)[0].cpu().numpy()
        f = lambda v: float((g * turned(v, pos, 12, interleaved, None, False)[0]).sum())
        for at in [(0, 0, 0), (1, 1, 5), (2, 0, 7), (2, 1, 15)]:
            e = np.zeros_like(x)
            e[at] = 1e-3
            assert abs((f(x + e) - f(x - e)) / 2e-3 - got[at]) < 1e-5      # f is linear: the difference is exact to 1e-12


def test_non_finite_values_stay_in_their_pairs():
    x = tt.ones((2, 1, 8), device="cuda", dtype=tt.float16)
    x[0, 0, 1], x[1, 0, 2] = float("inf"), float("nan")
    y = tqa.Rotary(8)(x, None, tt.tensor([3, 4], device="cuda"))[0]
    bad = ~tt.isfinite(y)
    assert bad.nonzero().tolist() == [[0, 0, 1], [0, 0, 5], [1, 0, 2], [1, 0, 6]]


def test_nothing_to_do_and_no_tokens():
    rot = tqa.Rotary(64)
    q, k = rot(tt.empty((0, 4, 64), device="cuda"), tt.empty((0, 0, 64), device="cuda"), tt.empty(0, dtype=tt.int64, device="cuda"))
    assert q.shape == (0, 4, 64) and k.shape == (0, 0, 64)


def test_captured_and_on_another_stream():
    gen = tt.Generator("cuda").manual_seed(6)
    q, k = (tt.randn((5, h, 128), generator=gen, device="cuda").half() for h in (8, 2))
    pos = tt.arange(5, device="cuda")
    rot = tqa.Rotary(128)
    out = tt.empty_like(q), tt.empty_like(k)
    side = tt.cuda.Stream()
    side.wait_stream(tt.cuda.current_stream())
    with tt.cuda.stream(side):
        rot(q, k, pos, out=out)
    tt.cuda.current_stream().wait_stream(side)
    graph = tt.cuda.CUDAGraph()
    with tt.cuda.graph(graph):
        rot(q, k, pos, out=out)
    for step in range(3):
        pos += 1000
        want = rot(q, k, pos)
        tt.cuda.synchronize()
        graph.replay()
        assert all(tt.equal(a, b) for a, b in zip(out, want))


def test_refusals():
    rot = tqa.Rotary(64)
    q, pos = tt.zeros((4, 2, 128), device="cuda"), tt.zeros(4, dtype=tt.int64, device="cuda")
    for call, error, text in [
            (lambda: rot(None, None, pos), ValueError, "neither"),
            (lambda: rot(q, q[:3], pos), ValueError, "same tokens"),
            (lambda: rot(q, q.half(), pos), ValueError, "same tokens"),
            (lambda: rot(q[0], None, pos), ValueError, r"\[tokens, heads"),
            (lambda: rot(q.double(), None, pos), TypeError, "float64"),
            (lambda: rot(q, None, pos[:3]), ValueError, "positions"),
            (lambda: rot(q, None, pos.float()), ValueError, "positions"),
            (lambda: rot(q.cpu(), None, pos), ValueError, "current device"),
            (lambda: rot(q, None, pos.cpu()), ValueError, "current device"),
            (lambda: rot(q.transpose(1, 2), None, pos), ValueError, "next to each other|rotary_dim"),
            (lambda: rot(q, None, pos, out=(q[:3], None)), ValueError, "out must"),
            (lambda: rot(q[..., :32].contiguous(), None, pos), ValueError, "rotary_dim 64"),
            (lambda: tqa.Rotary(2048)(tt.zeros((1, 1, 2048), device="cuda"), None, pos[:1]), NotImplementedError, "1024")]:
        with pytest.raises(error, match=text):
            call()
