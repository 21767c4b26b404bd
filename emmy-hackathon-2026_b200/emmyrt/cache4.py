"""A paged key / value cache in 4 bits: appending tokens to it, and attention over it.

A token's vector of one head is held as levels 0 .. 15 with an f16 step and least value: an element
stands for ``level * step + least``.  At head dim 128 that is 68 bytes instead of the 256 of bf16.
"""

from __future__ import annotations

import ctypes
import math

from . import Cache4AppendArgs, Cache4AttendArgs, DeviceBuffer, EmmyRTError, check, lib, ops_lib
from .operands import CODE, FLOATS, INDICES, Array, Operator, apart, contiguous, f32, operand, overlaps, shaped, written

DIMS = (64, 128)


class Cache4(Operator):
    """Pages of ``page`` token rows each, shared by all sequences; a slot is ``page index * page + row``.

    ``k`` and ``v`` are u8 [pages, heads, page, dim / 2] (element 2 i in the low half of byte i), ``k_meta`` and
    ``v_meta`` f16 [pages, heads, page, 2] (step, least).  :meth:`allocate` makes them.
    """

    def __init__(self, k, k_meta, v, v_meta):
        super().__init__()
        d = self.device
        self.k = contiguous(operand(k, "k", ("u8",), 4, d), "k")
        self.pages, self.heads, self.page, half = self.k.shape
        self.dim = 2 * half
        if self.dim not in DIMS:
            raise ValueError(f"head dim {self.dim} is not one of {DIMS}")
        self.v = shaped(contiguous(operand(v, "v", ("u8",), 4, d), "v"), "v", self.k.shape)
        meta = (self.pages, self.heads, self.page, 2)
        self.k_meta = shaped(contiguous(operand(k_meta, "k_meta", ("f16",), 4, d), "k_meta"), "k_meta", meta)
        self.v_meta = shaped(contiguous(operand(v_meta, "v_meta", ("f16",), 4, d), "v_meta"), "v_meta", meta)
        arrays = self.arrays = (self.k, self.v, self.k_meta, self.v_meta)
        for i, p in enumerate(arrays):
            for q in arrays[:i]:
                apart(p, q, "a part of the cache", same=False)

    @classmethod
    def allocate(cls, pages: int, heads: int, page: int, dim: int) -> "Cache4":
        """A cache in new device memory, all of it zero when this returns."""
        made = []
        for dtype, last, size in (("u8", dim // 2, 1), ("f16", 2, 2)) * 2:
            buffer = DeviceBuffer(pages * heads * page * last * size)
            buffer.zero()
            made.append(Array(buffer, dtype, (pages, heads, page, last)))
        # the streams that append need not wait for the default one
        check(lib.emmy_rt_stream_synchronize(0), "sync")
        return cls(*made)

    def _held(self) -> dict:
        return dict(cache_k=self.k.ptr, cache_v=self.v.ptr, cache_k_meta=self.k_meta.ptr, cache_v_meta=self.v_meta.ptr,
                    cache_pages=self.pages, cache_heads=self.heads, cache_page=self.page, cache_dim=self.dim)

    def append(self, k, v, slots, *, k_stored=None, v_stored=None, stream: int = 0) -> None:
        """Quantises ``k`` and ``v`` [tokens, heads, dim] into ``slots`` [tokens] (int32 or int64).  A token whose slot is
        negative or past the cache is left out (padding); two tokens of one call must not have the same slot.
        ``k_stored`` / ``v_stored`` receive the values that the cache then stands for, in the operands' type."""
        self._call((k, v, slots, k_stored, v_stored), None, stream)

    _FIELDS = ("k", "v", "slots", "k_stored", "v_stored")

    def _plan(self, operands, options) -> tuple:
        k, v, slots, k_stored, v_stored = operands
        d = self.device
        k = operand(k, "k", FLOATS, 3, d)
        n = k.shape[0]
        shaped(k, "k", (n, self.heads, self.dim))
        v = shaped(operand(v, "v", (k.dtype,), 3, d), "v", k.shape)
        slots = shaped(operand(slots, "slots", INDICES, 1, d), "slots", (n,))
        a = Cache4AppendArgs(**self._held(), k_token=k.strides[0], k_head=k.strides[1], v_token=v.strides[0],
                             v_head=v.strides[1], tokens=n, slots_64=slots.dtype == "i64", dtype=CODE[k.dtype])
        ins, outs = [(0, k, "k"), (1, v, "v"), (2, slots, "slots")], []
        for place, name, out in ((3, "k_stored", k_stored), (4, "v_stored", v_stored)):
            if out is not None:
                outs.append((place, contiguous(shaped(operand(out, name, (k.dtype,), 3, d), name, k.shape), name), name))
        held = [(5 + i, part, "the cache") for i, part in enumerate(self.arrays)]
        checks = overlaps(outs, ins)
        for part in held:
            checks += overlaps([part], ins + outs)
        return "emmy_ops_cache4_append", a, self._FIELDS, checks, self.arrays


class Cache4Attention(Operator):
    """Attention of ``q_heads`` query heads over a :class:`Cache4`; ``q_heads / cache.heads`` of them share a cached head.

    The object owns the workspace of its calls: calls of one object must not overlap on the GPU (one stream, or events;
    graphs that hold them likewise).  Make one for each stream that runs at the same time as others.
    """

    def __init__(self, cache: Cache4, q_heads: int):
        super().__init__()
        if cache.device != self.device:
            raise ValueError(f"the cache is on GPU {cache.device}, the current one is {self.device}")
        if q_heads < 1 or q_heads % cache.heads:
            raise ValueError(f"{q_heads} query heads over {cache.heads} heads of the cache")
        self.cache, self.q_heads = cache, int(q_heads)
        need = ctypes.c_uint64()
        status = ops_lib().emmy_ops_cache4_attend_workspace(cache.dim, self.device, ctypes.byref(need))
        if status:
            raise EmmyRTError(status, "attention workspace", ops_lib().emmy_ops_last_error().decode(errors="replace"))
        self._workspace = DeviceBuffer(need.value)

    def __call__(self, q, out, table, lengths, *, scale: float | None = None, stream: int = 0) -> None:
        """``q`` and ``out`` are [batch, tokens, q_heads, dim] (f16 or bf16), ``lengths`` [batch] and ``table``
        [batch, pages] int32: position p of sequence b is row ``p % page`` of the cache's page ``table[b, p // page]``.
        Query i stands at position ``lengths[b] - tokens + i`` (its key is in the cache already) and sees the positions up
        to its own; a query that sees nothing gives zeros.  Lengths beyond the table are cut there; pages that are none
        are not seen.  ``scale`` is 1 / sqrt(dim) by default.  ``out`` may be ``q``."""
        scale = self.cache.dim ** -0.5 if scale is None else float(scale)
        self._call((q, out, table, lengths), scale, stream)

    _FIELDS = ("q", "out", "table", "lengths")

    def _plan(self, operands, scale) -> tuple:
        q, out, table, lengths = operands
        c, d = self.cache, self.device
        if not f32(scale / math.log(2.0)):          # the kernel's logits are to base 2
            raise ValueError(f"scale {scale}")
        q = operand(q, "q", ("f16", "bf16"), 4, d)
        batch, tokens = q.shape[:2]
        shaped(q, "q", (batch, tokens, self.q_heads, c.dim))
        out = written(shaped(operand(out, "out", (q.dtype,), 4, d), "out", q.shape), "out")
        table = operand(table, "table", ("i32",), 2, d)
        if table.shape[0] != batch:
            raise ValueError(f"table has {table.shape[0]} rows for {batch} sequences")
        lengths = shaped(operand(lengths, "lengths", ("i32",), 1, d), "lengths", (batch,))
        a = Cache4AttendArgs(**c._held(), workspace=self._workspace.ptr, workspace_bytes=self._workspace.nbytes,
                             q_batch=q.strides[0], q_token=q.strides[1], q_head=q.strides[2], out_batch=out.strides[0],
                             out_token=out.strides[1], out_head=out.strides[2], table_stride=table.strides[0], batch=batch,
                             tokens=tokens, q_heads=self.q_heads, max_pages=table.shape[1], dtype=CODE[q.dtype], scale=scale)
        others = [(0, q, "q"), (2, table, "table"), (3, lengths, "lengths")]
        others += [(4 + i, part, "the cache") for i, part in enumerate(c.arrays)]
        return "emmy_ops_cache4_attend", a, self._FIELDS, overlaps([(1, out, "out")], others, same=((1, 0),)), c.arrays
