"""Norms before and after a block of a residual network, with its gate and residual scale, in one pass.

The compiler's row reductions cover a norm on its own (``x_l_rmsnorm_w``, ``x_f_layernorm``); a
network runs two of them around every block, with the residual sum between: this operator reads the
residual stream and the block's output once and writes the new stream and the next block's input.
"""

from __future__ import annotations

from . import NormArgs
from .operands import CODE, FLOATS, Operator, f32, operand, overlaps, shaped, written

KINDS = {"rms": 0, "layer": 1}
MAX_DIM = 16384


class ResidualNorm(Operator):
    """``y = x + scale * gate * N(block)``, ``h = N(y)`` over rows of ``dim`` elements.

    ``N`` is an RMS norm (``kind="rms"``) or a layer norm (``"layer"``) with its own weight and bias on
    either side; ``post_norm=False`` leaves ``block`` as it is.  Everything between the operands is
    computed in f32; ``h`` is taken of ``y`` before ``y`` is rounded.
    """

    def __init__(self, dim: int, kind: str = "rms", eps: float = 1e-6, scale: float = 1.0, post_norm: bool = True):
        if kind not in KINDS:
            raise ValueError(f"kind {kind!r} is not one of {', '.join(KINDS)}")
        if not 1 <= dim <= MAX_DIM:
            raise ValueError(f"dim {dim} is not in 1 .. {MAX_DIM}")
        if not (eps >= 0 and f32(eps)):
            raise ValueError(f"eps {eps}")
        if not f32(scale):
            raise ValueError(f"scale {scale}")
        self.dim, self.kind, self.eps, self.scale, self.post_norm = int(dim), kind, float(eps), float(scale), bool(post_norm)
        super().__init__()

    def __call__(self, x, block, y, h=None, *, post_weight=None, post_bias=None, gate=None, rows_per_gate: int | None = None,
                 pre_weight=None, pre_bias=None, stream: int = 0) -> None:
        """``x``, ``block``, ``y`` and ``h`` are [rows, dim] of one type (f32, f16 or bf16); ``y`` may be ``x`` and
        ``h`` may be ``block``.  Weights and biases are [dim] of any of the three types, ``gate`` [gates, dim]: row
        ``r`` takes gate row ``r // rows_per_gate`` (all rows the first one where it is not given)."""
        self._call((x, block, y, h, post_weight, post_bias, gate, pre_weight, pre_bias), rows_per_gate, stream)

    _FIELDS = ("x", "block", "y", "h", "post_weight", "post_bias", "gate", "pre_weight", "pre_bias")

    def _plan(self, operands, rows_per_gate) -> tuple:
        x, block, y, h, post_weight, post_bias, gate, pre_weight, pre_bias = operands
        d = self.device
        x = operand(x, "x", FLOATS, 2, d)
        rows, dim = x.shape
        if dim != self.dim:
            raise ValueError(f"x has {dim} columns, the operator {self.dim}")
        block = shaped(operand(block, "block", (x.dtype,), 2, d), "block", x.shape)
        y = written(shaped(operand(y, "y", (x.dtype,), 2, d), "y", x.shape), "y")
        a = NormArgs(x_stride=x.strides[0], block_stride=block.strides[0], y_stride=y.strides[0], rows=rows, dim=dim,
                     dtype=CODE[x.dtype], kind=KINDS[self.kind], post_norm=self.post_norm, eps=self.eps, scale=self.scale,
                     rows_per_gate=max(1, rows))
        if h is not None:
            h = written(shaped(operand(h, "h", (x.dtype,), 2, d), "h", x.shape), "h")
            a.h_stride = h.strides[0]
        elif pre_weight is not None or pre_bias is not None:
            raise ValueError("pre_weight and pre_bias are of h, which is not asked for")
        if not self.post_norm and (post_weight is not None or post_bias is not None):
            raise ValueError("post_weight and post_bias are of the norm that post_norm=False leaves out")
        vectors = []
        for place, name, v in ((4, "post_weight", post_weight), (5, "post_bias", post_bias), (7, "pre_weight", pre_weight),
                               (8, "pre_bias", pre_bias)):
            if v is not None:
                v = shaped(operand(v, name, FLOATS, 1, d), name, (dim,))
                setattr(a, name + "_dtype", CODE[v.dtype])
                vectors.append((place, v, name))
        if rows_per_gate is not None and rows_per_gate < 1:
            raise ValueError(f"rows_per_gate {rows_per_gate}")
        if gate is not None:
            gate = operand(gate, "gate", FLOATS, 2, d)
            per = max(1, rows) if rows_per_gate is None else int(rows_per_gate)
            if gate.shape[1] != dim or gate.shape[0] * per < rows:
                raise ValueError(f"gate of shape {tuple(gate.shape)} for {rows} rows, {per} each, of {dim}")
            a.gate_dtype, a.gate_stride, a.rows_per_gate = CODE[gate.dtype], gate.strides[0], per
            vectors.append((6, gate, "gate"))
        checks = overlaps([(2, y, "y"), (3, h, "h")], [(0, x, "x"), (1, block, "block"), *vectors],
                          same=((2, 0), (2, 1), (3, 0), (3, 1)))
        return "emmy_ops_residual_norm", a, self._FIELDS, checks
