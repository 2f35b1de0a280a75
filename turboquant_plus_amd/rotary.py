"""Rotary positions: queries and keys turned by angles that grow with their position, before the keys enter a cache.

No counterpart in the reference, whose keys arrive rotated (tests/test_kv_cache.py:73-89 attends to the rows as they are).
Pair i of the first `rotary_dim` values of a head is turned by position * frequency_i, frequency_i = base^(-2i / rotary_dim),
changed by `RotaryScaling` for contexts longer than a model was trained on.
"""
from __future__ import annotations

import ctypes as C
import math
from dataclasses import dataclass

import numpy as np

from . import _lib as L

SCALINGS = ("linear", "ntk", "yarn")


@dataclass(frozen=True)
class RotaryScaling:
    """How frequencies are changed for a context `factor` times as long.

    linear: all frequencies divided by the factor (position interpolation).
    ntk:    the base raised by factor^(r / (r - 2)), which divides the slowest frequency by the factor and keeps the fastest.
    yarn:   by parts: pairs that turn `fast_turns` times or more over `trained_tokens` keep their frequency, those that turn
            `slow_turns` times or less have it divided, with a linear ramp over the pairs' numbers between; the turned
            values are multiplied by `magnitude` (default 0.1 ln(factor) + 1).
    """
    kind: str
    factor: float
    trained_tokens: int | None = None
    fast_turns: float = 32.0
    slow_turns: float = 1.0
    magnitude: float | None = None

    def __post_init__(self):
        if self.kind not in SCALINGS:
            raise ValueError(f"scaling must be one of {SCALINGS}, got {self.kind!r}")
        if not self.factor > 0 or not math.isfinite(self.factor):
            raise ValueError(f"factor must be positive, got {self.factor}")
        if self.kind == "yarn" and (self.trained_tokens is None or self.trained_tokens < 1):
            raise ValueError("yarn needs trained_tokens, the context length that the frequencies were trained on")
        if not 0 < self.slow_turns <= self.fast_turns:
            raise ValueError("slow_turns must be positive and at most fast_turns")


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: RotaryScaling | None = None) -> tuple[np.ndarray, float]:
    """(radians per position of each pair in float64, what the turned values are multiplied by)."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if not base > 1 or not math.isfinite(base):
        raise ValueError(f"base must be over 1, got {base}")
    i = np.arange(rotary_dim // 2, dtype=np.float64)
    if scaling is not None and scaling.kind == "ntk":
        if rotary_dim == 2:
            raise ValueError("ntk scaling needs a rotary_dim of 4 or more")
        base = base * scaling.factor ** (rotary_dim / (rotary_dim - 2))
    f = base ** (-2.0 * i / rotary_dim)
    if scaling is None or scaling.kind == "ntk":
        return f, 1.0
    if scaling.kind == "linear":
        return f / scaling.factor, 1.0
    # the pair that turns `turns` times over the trained tokens
    pair = lambda turns: rotary_dim * math.log(scaling.trained_tokens / (turns * 2 * math.pi)) / (2 * math.log(base))
    lo = max(math.floor(pair(scaling.fast_turns)), 0)
    hi = min(math.ceil(pair(scaling.slow_turns)), rotary_dim - 1)
    ramp = np.clip((i - lo) / max(hi - lo, 1e-3), 0.0, 1.0)
    magnitude = 0.1 * math.log(scaling.factor) + 1.0 if scaling.magnitude is None else float(scaling.magnitude)
    return f * (1 - ramp) + f / scaling.factor * ramp, magnitude


class Rotary:
    """Turns queries and keys to their positions in one launch (tq_rotary).

    interleaved: pairs are neighbouring values (2i, 2i + 1); otherwise i and i + rotary_dim / 2.
    Values of a head beyond rotary_dim stay as they are.  The object holds the frequencies on the current device.
    """

    def __init__(self, rotary_dim: int, *, base: float = 10000.0, interleaved: bool = False, scaling: RotaryScaling | None = None):
        f, self.magnitude = rotary_frequencies(rotary_dim, base, scaling)
        self.rotary_dim, self.interleaved = rotary_dim, bool(interleaved)
        self.turns = L.torch().from_numpy(f / (2 * math.pi)).to(L.require_gpu())

    def __call__(self, q, k, positions, *, inverse: bool = False, out=None):
        """q [tokens, query heads, head_dim] and k [tokens, KV heads, head_dim] (either may be None) in float16, bfloat16 or
        float32, of any strides with a head's values next to each other; positions [tokens], int32 or int64 -> (q, k) turned, new
        tensors or `out`: a pair of tensors of those shapes, which may be (q, k) themselves.
        inverse: turned back; with it a gradient with respect to the turned tensors becomes that of the given ones."""
        tt = L.torch()
        some = q if q is not None else k
        if some is None:
            raise ValueError("neither q nor k")
        dtype, device = some.dtype, L._current_device()
        code = _DTYPES.get(dtype)
        if code is None:
            _DTYPES.update({tt.float16: L.TQ_F16, tt.float32: L.TQ_F32, tt.bfloat16: L.TQ_BF16})
            code = _DTYPES.get(dtype)
        tokens, dim = some.shape[0], some.shape[-1]
        for x in (q, k):
            if x is not None and (len(x.shape) != 3 or x.shape[0] != tokens or x.shape[2] != dim or x.dtype is not dtype):
                raise ValueError("q and k must be [tokens, heads, head_dim] with the same tokens, head_dim and dtype")
        if out is None:
            out = None if q is None else q.new_empty(q.shape), None if k is None else k.new_empty(k.shape)
        elif len(out) != 2 or any((x is None) != (o is None) or (o is not None and (o.shape != x.shape or o.dtype != dtype))
                                  for x, o in zip((q, k), out)):
            raise ValueError("out must be a pair of tensors of q's and k's shapes and dtype")
        index = positions.dtype
        if (index is not tt.int32 and index is not tt.int64) or positions.shape != (tokens,):
            raise ValueError("positions must be int32 or int64 [tokens]")
        if not positions.is_contiguous():
            positions = positions.contiguous()
        # (heads, strides and address of q and its output, then of k)
        sides = []
        for x, o in ((q, out[0]), (k, out[1])):
            if x is None:
                sides.append((0, 0, 0, 0, 0, None, None))
                continue
            if x.get_device() != device or o.get_device() != device:
                raise ValueError(_PLACE)
            (a, b, c), (d, e, f) = x.stride(), o.stride()
            if dim > 1 and (c != 1 or f != 1):
                raise ValueError("a head's values must be next to each other")
            sides.append((x.shape[1], a, b, d, e, x.data_ptr(), o.data_ptr()))
        if positions.get_device() != device or self.turns.get_device() != device:
            raise ValueError(_PLACE)
        if code is None:
            raise TypeError(f"unsupported dtype {dtype}")
        (hq, qa, qb, oa, ob, q_at, oq_at), (hk, ka, kb, pa, pb, k_at, ok_at) = sides
        p = L.TQRotaryParams(tokens, hq, hk, dim, self.rotary_dim, self.interleaved, inverse, code, index is tt.int64, self.magnitude, qa, qb,
                             ka, kb, oa, ob, pa, pb)
        L.check(L.lib().tq_rotary(C.byref(p), q_at, oq_at, k_at, ok_at, positions.data_ptr(), self.turns.data_ptr(), L.stream_ptr()))
        return out


_DTYPES = {}      # torch dtype -> its code
_PLACE = "q, k, positions and the frequencies must be on the current device"
