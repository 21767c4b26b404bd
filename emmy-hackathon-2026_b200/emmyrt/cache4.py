"""A paged key / value cache in 4 bits: appending tokens to it.

A token's vector of one head is held as levels 0 .. 15 with an f16 step and least value: an element
stands for ``level * step + least``.  At head dim 128 that is 68 bytes instead of the 256 of bf16.
"""

from __future__ import annotations

from . import Cache4AppendArgs, Cache4Memory, DeviceBuffer
from .operands import (CODE, FLOATS, INDICES, Array, apart, call, contiguous, operand, own_device, shaped)

DIMS = (64, 128)


class Cache4:
    """Pages of ``page`` token rows each, shared by all sequences; a slot is ``page index * page + row``.

    ``k`` and ``v`` are u8 [pages, heads, page, dim / 2] (element 2 i in the low half of byte i), ``k_meta`` and
    ``v_meta`` f16 [pages, heads, page, 2] (step, least).  :meth:`allocate` makes them.
    """

    def __init__(self, k, k_meta, v, v_meta):
        self.device = d = own_device()
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
        """A cache in new device memory, all of it zero."""
        made = []
        for dtype, last, size in (("u8", dim // 2, 1), ("f16", 2, 2)) * 2:
            buffer = DeviceBuffer(pages * heads * page * last * size)
            buffer.zero()
            made.append(Array(buffer, dtype, (pages, heads, page, last)))
        return cls(*made)

    def memory(self) -> Cache4Memory:
        return Cache4Memory(k=self.k.ptr, v=self.v.ptr, k_meta=self.k_meta.ptr, v_meta=self.v_meta.ptr, pages=self.pages,
                            heads=self.heads, page=self.page, dim=self.dim)

    def append(self, k, v, slots, *, k_stored=None, v_stored=None, stream: int = 0) -> None:
        """Quantises ``k`` and ``v`` [tokens, heads, dim] into ``slots`` [tokens] (int32 or int64).  A token whose slot is
        negative or past the cache is left out (padding); two tokens of one call must not have the same slot.
        ``k_stored`` / ``v_stored`` receive the values that the cache then stands for, in the operands' type."""
        d = self.device
        k = operand(k, "k", FLOATS, 3, d)
        n = k.shape[0]
        shaped(k, "k", (n, self.heads, self.dim))
        v = shaped(operand(v, "v", (k.dtype,), 3, d), "v", k.shape)
        slots = shaped(operand(slots, "slots", INDICES, 1, d), "slots", (n,))
        a = Cache4AppendArgs(cache=self.memory(), k=k.ptr, v=v.ptr, slots=slots.ptr, k_token=k.strides[0],
                             k_head=k.strides[1], v_token=v.strides[0], v_head=v.strides[1], tokens=n,
                             slots_64=slots.dtype == "i64", dtype=CODE[k.dtype])
        outs = []
        for name, out in (("k_stored", k_stored), ("v_stored", v_stored)):
            if out is not None:
                out = contiguous(shaped(operand(out, name, (k.dtype,), 3, d), name, k.shape), name)
                if out.ptr % 16:
                    raise ValueError(f"{name} does not start on 16 bytes")
                setattr(a, name, out.ptr)
                for other in (*outs, k, v, slots, *self.arrays):
                    apart(out, other, name, same=False)
                outs.append(out)
        for part in self.arrays:
            for other in (k, v, slots):
                apart(part, other, "an operand", same=False)
        call("emmy_ops_cache4_append", a, d, stream)
