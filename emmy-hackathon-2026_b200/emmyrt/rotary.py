"""Rotary positions from their angles.

The compiler's element maps rotate by cosines and sines that the caller has (``x_l_rope``); this
operator computes them from positions, once per token for all heads, with the scalings of the
frequencies that long contexts use.
"""

from __future__ import annotations

import math

import numpy as np

from . import DeviceBuffer, RotaryArgs
from .operands import CODE, FLOATS, INDICES, Operator, f32, operand, overlaps, shaped, written

LAYOUTS = {"half": 0, "interleaved": 1}
SCALINGS = ("none", "linear", "base", "parts")


def frequencies(rotary_dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                original_length: int = 4096, slow: float = 1.0, fast: float = 32.0) -> np.ndarray:
    """Radians per position of each pair, in f64: ``base ** (-2 i / rotary_dim)``, and for contexts ``factor``
    times as long

    * ``linear``: all divided by ``factor`` (positions interpolated);
    * ``base``: the base raised by ``factor ** (d / (d - 2))``, which leaves the fastest pair and divides the slowest
      one by ``factor``;
    * ``parts``: pairs that turn at least ``fast`` times within ``original_length`` are left, those that turn at most
      ``slow`` times are divided by ``factor``, those between are mixed linearly in their number of turns.
    """
    d = rotary_dim
    if d < 2 or d % 2:
        raise ValueError(f"rotary_dim {d} is not a positive even number")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling {scaling!r} is not one of {', '.join(SCALINGS)}")
    if not (base > 0 and math.isfinite(base)) or not (factor > 0 and math.isfinite(factor)):
        raise ValueError(f"base {base}, factor {factor}")
    if scaling == "base":
        if d == 2:
            raise ValueError("a single pair has no base to raise")
        base = base * factor ** (d / (d - 2))
    f = base ** (-np.arange(0, d, 2, dtype=np.float64) / d)
    if scaling == "linear":
        f = f / factor
    elif scaling == "parts":
        if original_length < 1 or not slow < fast:
            raise ValueError(f"original_length {original_length}, slow {slow}, fast {fast}")
        keep = np.clip((original_length * f / (2 * math.pi) - slow) / (fast - slow), 0.0, 1.0)
        f = f / factor * (1 - keep) + f * keep
    return f


class Rotary(Operator):
    """Rotates the first ``rotary_dim`` elements of each head of ``dim``; the others are copied.

    ``layout="half"`` pairs element i with i + rotary_dim / 2, ``"interleaved"`` 2 i with 2 i + 1.  Pairs are
    multiplied by ``magnitude`` too (by default 1, and 0.1 ln(factor) + 1 with ``scaling="parts"``).  Angles are
    kept in turns as 64-bit fractions, so far positions are as exact as near ones.
    """

    def __init__(self, dim: int, rotary_dim: int | None = None, base: float = 10000.0, layout: str = "half",
                 scaling: str = "none", factor: float = 1.0, original_length: int = 4096, slow: float = 1.0,
                 fast: float = 32.0, magnitude: float | None = None):
        rotary_dim = dim if rotary_dim is None else rotary_dim
        if layout not in LAYOUTS:
            raise ValueError(f"layout {layout!r} is not one of {', '.join(LAYOUTS)}")
        if not 2 <= rotary_dim <= dim <= 8192:
            raise ValueError(f"rotary_dim {rotary_dim} of dim {dim}")
        f = frequencies(rotary_dim, base, scaling, factor, original_length, slow, fast)
        if magnitude is None:
            magnitude = 0.1 * math.log(factor) + 1.0 if scaling == "parts" else 1.0
        if not f32(magnitude):
            raise ValueError(f"magnitude {magnitude}")
        self.dim, self.rotary_dim, self.layout, self.magnitude = int(dim), int(rotary_dim), layout, float(magnitude)
        super().__init__()
        # whole turns do nothing: the fraction in 64 bits (53 of them known)
        turns = np.array([int((v / (2 * math.pi)) % 1.0 * 2.0 ** 64) for v in f.tolist()], dtype=np.uint64)
        self._turns = DeviceBuffer(turns.nbytes)
        self._turns.upload(turns)

    def __call__(self, positions, q, k=None, *, q_out=None, k_out=None, inverse: bool = False, stream: int = 0) -> None:
        """``q`` (and ``k``, in the same launch) are [tokens, heads, dim], of one type;
        ``positions`` [tokens] int32 or int64.  ``q_out`` / ``k_out`` receive them; without one its operand is rotated in
        place.  ``inverse`` turns the other way: the gradient of the rotation (and its inverse where magnitude is 1)."""
        self._call((positions, q, k, q if q_out is None else q_out, k if k_out is None else k_out), bool(inverse), stream)

    _FIELDS = ("positions", "x0", "x1", "out0", "out1")

    def _plan(self, operands, inverse) -> tuple:
        d = self.device
        positions = operand(operands[0], "positions", INDICES, 1, d)
        n = positions.shape[0]
        a = RotaryArgs(turns=self._turns.ptr, tokens=n, positions_64=positions.dtype == "i64", dim=self.dim,
                       rotary=self.rotary_dim, layout=LAYOUTS[self.layout], transpose=inverse, magnitude=self.magnitude)
        if operands[2] is None and operands[4] is not None:
            raise ValueError("k_out without k")
        dtype, ins, outs = None, [(0, positions, "positions")], []
        for i, name in enumerate(("q", "k")):
            if i and operands[2] is None:
                continue
            v = operand(operands[1 + i], name, FLOATS if dtype is None else (dtype,), 3, d)
            dtype = v.dtype
            if v.shape[0] != n or v.shape[2] != self.dim:
                raise ValueError(f"{name} has shape {tuple(v.shape)}, wanted ({n}, heads, {self.dim})")
            o = shaped(operand(operands[3 + i], name + "_out", (dtype,), 3, d), name + "_out", v.shape)
            written(o, name + "_out")
            setattr(a, f"heads{i}", v.shape[1])
            for field, stride in (("x_token", v.strides[0]), ("x_head", v.strides[1]), ("out_token", o.strides[0]),
                                  ("out_head", o.strides[1])):
                setattr(a, f"{field}{i}", stride)
            ins.append((1 + i, v, name))
            outs.append((3 + i, o, name + "_out"))
        a.dtype = CODE[dtype]
        return "emmy_ops_rotary", a, self._FIELDS, overlaps(outs, ins, same=((3, 1), (4, 2)))
