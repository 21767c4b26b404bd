"""FP8 (e4m3) linear maps with a scale for each block of 128.

:mod:`emmyrt.fp8` scales a whole matrix by its largest element; here every row of x has a scale for each
128 columns and W one for each 128 x 128 block, so one loud channel costs its own block only.  The scales are
f32 numbers, ``amax / 448`` (1 where a block is zero); quantised values are ``e4m3(v / scale)``.
"""

from __future__ import annotations

import numpy as np

from . import BlockFp8LinearArgs, BlockFp8QuantizeArgs, DeviceBuffer, check, current_device, lib
from .operands import CODE, FLOATS, Array, Operator, operand, overlaps, shaped, written

BLOCK = 128


def pitch(cols: int) -> int:
    """Bytes from row to row of a quantised matrix: rows start on 16 bytes."""
    return -(-cols // 16) * 16


def blocks(extent: int) -> int:
    return -(-extent // BLOCK)


class BlockFp8Quantizer(Operator):
    """``q = e4m3(x / s)`` with a scale for each row and 128 columns, or (``square``) each 128 x 128 block."""

    def __init__(self, square: bool = False):
        super().__init__()
        self.square = bool(square)

    def __call__(self, x, q, s, *, stream: int = 0) -> None:
        """``x`` [rows, cols] (f32, f16 or bf16); ``q`` the same shape, e4m3 or u8, its rows a multiple of 16 bytes apart and
        at least :func:`pitch` (without ``square`` the columns up to there become zero, those of the last row too; a
        single row that is not that far apart has no such columns); ``s`` f32 [blocks of cols, rows], with ``square``
        [blocks of rows, blocks of cols]."""
        if not self.square:
            _room_for_padding(q)
        self._call((x, q, s), None, stream)

    def _plan(self, operands, options) -> tuple:
        d = self.device
        x = operand(operands[0], "x", FLOATS, 2, d)
        rows, cols = x.shape
        if cols < 1:
            raise ValueError("x has no columns")
        q = written(shaped(operand(operands[1], "q", ("e4m3", "u8"), 2, d), "q", x.shape), "q")
        q = _padded(q, "q")
        want = (blocks(rows), blocks(cols)) if self.square else (blocks(cols), rows)
        s = written(shaped(operand(operands[2], "s", ("f32",), 2, d), "s", want), "s")
        a = BlockFp8QuantizeArgs(x_stride=x.strides[0], q_stride=_stride(q) if self.square else _row_stride(q),
                                 s_stride=s.strides[0], rows=rows, cols=cols,
                                 dtype=CODE[x.dtype], square=self.square)
        checks = overlaps([(1, _with_padding(q) if not self.square else q, "q"), (2, s, "s")], [(0, x, "x")])
        return "emmy_ops_blockfp8_quantize", a, ("x", "q", "s"), checks


def _padded(q: Array, name: str) -> Array:
    if q.shape[0] > 1 and (q.strides[0] % 16 or q.strides[0] < pitch(q.shape[1])):
        raise ValueError(f"{name}: rows are {q.strides[0]} bytes apart, wanted a multiple of 16 from {pitch(q.shape[1])} on")
    return q


def _stride(q: Array) -> int:
    """The row stride; a single row has none of its own."""
    return q.strides[0] if q.shape[0] > 1 else pitch(q.shape[1])


def _row_stride(q: Array) -> int:
    """The row stride for the row quantiser, which pads what it allows: a single row that is not in padded rows has none."""
    rows, cols = q.shape
    apart = q.strides[0]
    return apart if rows > 1 or (apart >= pitch(cols) and apart % 16 == 0) else cols


def _with_padding(q: Array) -> Array:
    """``q`` with the columns that the row quantiser fills with zeros."""
    stride = _row_stride(q)
    return Array(q.ptr, q.dtype, (q.shape[0], min(stride, pitch(q.shape[1]))), (stride, 1), q.device)


def _room_for_padding(q) -> None:
    """Refuses a q whose last row's padding lies past its memory, as far as that is known.  It is no matter of the call's
    kind, so each call asks."""
    if type(q) is Array:
        room, strides = getattr(q.owner, "nbytes", None), q.strides
    elif hasattr(q, "untyped_storage"):
        room, strides = q.untyped_storage().nbytes() - q.storage_offset(), q.stride()     # elements of one byte
    else:
        return
    if room is None or len(q.shape) != 2 or q.shape[1] % 16 == 0:
        return
    rows, cols = q.shape
    if rows and (rows > 1 or (strides[0] >= pitch(cols) and strides[0] % 16 == 0)) and \
            (rows - 1) * strides[0] + pitch(cols) > room:
        raise ValueError(f"q: the last row's padding, up to {pitch(cols)} columns, lies past its memory")


class BlockFp8Linear(Operator):
    """``y = x W^T``: x is quantised on the way, W [n, k] is given quantised (``wq`` e4m3 or u8, ``ws`` f32
    [blocks of n, blocks of k]).  Sums are f32; up to ``max_rows`` rows of x a call.

    The object owns the quantised x of its calls, so calls of one object must not overlap on the GPU (one stream, or
    events; graphs that hold them likewise).
    """

    def __init__(self, wq, ws, max_rows: int):
        super().__init__()
        d = self.device
        self.wq = _padded(operand(wq, "wq", ("e4m3", "u8"), 2, d), "wq")
        self.n, self.k = self.wq.shape
        if self.n < 1 or self.k < 1:
            raise ValueError(f"W of {self.n} x {self.k}")
        if self.wq.ptr % 16:
            raise ValueError("wq does not start on 16 bytes")
        self.ws = shaped(operand(ws, "ws", ("f32",), 2, d), "ws", (blocks(self.n), blocks(self.k)))
        if not 1 <= max_rows < 1 << 31:
            raise ValueError(f"max_rows {max_rows}")
        self.max_rows = int(max_rows)
        # the quantised x, its scales and the status word
        x_bytes = -(-self.max_rows * pitch(self.k) // 256) * 256
        self._xs_stride = -(-self.max_rows // 4) * 4
        s_bytes = -(-blocks(self.k) * self._xs_stride * 4 // 256) * 256
        # parts of a product that is cut along k: few rows of y at a time, so 16 MB hold every cut that pays
        self._parts_bytes = 0 if self.max_rows <= 8 else min(16 << 20, 16 * min(self.max_rows, 1024) * (self.n + 3) * 4)
        self._workspace = DeviceBuffer(x_bytes + s_bytes + 256 + self._parts_bytes)
        at = self._workspace.ptr
        self._xq, self._xs, self._status = at, at + x_bytes, at + x_bytes + s_bytes
        self._parts = self._status + 256
        self._clear_status()

    @classmethod
    def from_weight(cls, w, max_rows: int, stream: int = 0) -> "BlockFp8Linear":
        """Quantises ``w`` [n, k] (f32, f16 or bf16) into memory of its own, on ``stream``, and waits for that: calls may
        come on any stream."""
        d = cls.__new__(cls)
        Operator.__init__(d)
        w = operand(w, "w", FLOATS, 2, d.device)
        n, k = w.shape
        if n < 1 or k < 1:
            raise ValueError(f"W of {n} x {k}")
        wq = Array(DeviceBuffer(n * pitch(k)), "u8", (n, k), (pitch(k), 1))
        ws = Array(DeviceBuffer(blocks(n) * blocks(k) * 4), "f32", (blocks(n), blocks(k)))
        BlockFp8Quantizer(square=True)(w, wq, ws, stream=stream)
        check(lib.emmy_rt_stream_synchronize(stream), "sync")
        d.__init__(wq, ws, max_rows)
        return d

    def _clear_status(self) -> None:
        check(lib.emmy_rt_memset(self._status, 0, 4, 0), "memset")
        check(lib.emmy_rt_stream_synchronize(0), "sync")

    def status(self, stream: int | None = None) -> int:
        """The calls' status word (0 = ok; non-zero = a bounded wait inside the kernel gave up and y is not valid).
        Waits for all work of the operator's device, or for ``stream`` alone where all calls came on it (or before it);
        a non-zero word is cleared, so no call may be on its way meanwhile."""
        out = np.zeros(1, np.uint32)
        before = current_device()
        check(lib.emmy_rt_set_device(self.device), "set device")        # a thread may have none yet
        try:
            if stream is None:
                check(lib.emmy_rt_synchronize(), "synchronize")
                stream = 0
            check(lib.emmy_rt_memcpy_dtoh(out.ctypes.data, self._status, 4, stream), "dtoh")
            check(lib.emmy_rt_stream_synchronize(stream), "sync")
            if out[0]:
                check(lib.emmy_rt_memset(self._status, 0, 4, stream), "memset")
                check(lib.emmy_rt_stream_synchronize(stream), "sync")
        finally:
            if before != self.device:
                check(lib.emmy_rt_set_device(before), "set device")
        return int(out[0])

    def __call__(self, x, y, *, stream: int = 0) -> None:
        """``x`` [rows, k] and ``y`` [rows, n], each f32, f16 or bf16."""
        self._call((x, y), None, stream)

    def _plan(self, operands, options) -> tuple:
        d = self.device
        x = operand(operands[0], "x", FLOATS, 2, d)
        rows = x.shape[0]
        if x.shape[1] != self.k:
            raise ValueError(f"x has {x.shape[1]} columns, W {self.k}")
        if rows > self.max_rows:
            raise ValueError(f"{rows} rows, the operator was made for {self.max_rows}")
        y = written(shaped(operand(operands[1], "y", FLOATS, 2, d), "y", (rows, self.n)), "y")
        a = BlockFp8LinearArgs(xq=self._xq, xs=self._xs, wq=self.wq.ptr, ws=self.ws.ptr, status=self._status,
                               parts=self._parts if self._parts_bytes else 0, parts_bytes=self._parts_bytes,
                               xq_stride=pitch(self.k), xs_stride=self._xs_stride, wq_stride=_stride(self.wq),
                               ws_stride=self.ws.strides[0], y_stride=y.strides[0], m=rows, n=self.n, k=self.k,
                               dtype=CODE[y.dtype], x_stride=x.strides[0], x_dtype=CODE[x.dtype])
        checks = overlaps([(1, y, "y")], [(0, x, "x"), (2, self.wq, "wq"), (3, self.ws, "ws")])
        return "emmy_ops_blockfp8_linear", a, ("x", "y"), checks, (self.wq, self.ws)
