"""A paged key / value cache in 4 bits: appending tokens to it.

A token's vector of one head is held as levels 0 .. 15 with an f16 step and least value: an element
stands for ``level * step + least``.  At head dim 128 that is 68 bytes instead of the 256 of bf16.
"""

from __future__ import annotations

from . import Cache4AppendArgs, DeviceBuffer
from .operands import CODE, FLOATS, INDICES, Array, Operator, Plan, apart, contiguous, operand, overlaps, shaped

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
        """A cache in new device memory, all of it zero."""
        made = []
        for dtype, last, size in (("u8", dim // 2, 1), ("f16", 2, 2)) * 2:
            buffer = DeviceBuffer(pages * heads * page * last * size)
            buffer.zero()
            made.append(Array(buffer, dtype, (pages, heads, page, last)))
        return cls(*made)

    def append(self, k, v, slots, *, k_stored=None, v_stored=None, stream: int = 0) -> None:
        """Quantises ``k`` and ``v`` [tokens, heads, dim] into ``slots`` [tokens] (int32 or int64).  A token whose slot is
        negative or past the cache is left out (padding); two tokens of one call must not have the same slot.
        ``k_stored`` / ``v_stored`` receive the values that the cache then stands for, in the operands' type."""
        self._call((k, v, slots, k_stored, v_stored, *self.arrays), None, stream)

    _FIELDS = ("k", "v", "slots", "k_stored", "v_stored", "cache_k", "cache_v", "cache_k_meta", "cache_v_meta")

    def _plan(self, operands, options) -> Plan:
        k, v, slots, k_stored, v_stored = operands[:5]
        d = self.device
        k = operand(k, "k", FLOATS, 3, d)
        n = k.shape[0]
        shaped(k, "k", (n, self.heads, self.dim))
        v = shaped(operand(v, "v", (k.dtype,), 3, d), "v", k.shape)
        slots = shaped(operand(slots, "slots", INDICES, 1, d), "slots", (n,))
        a = Cache4AppendArgs(cache_pages=self.pages, cache_heads=self.heads, cache_page=self.page, cache_dim=self.dim,
                             k_token=k.strides[0], k_head=k.strides[1], v_token=v.strides[0],
                             v_head=v.strides[1], tokens=n, slots_64=slots.dtype == "i64", dtype=CODE[k.dtype])
        ins, outs = [(0, k, "k"), (1, v, "v"), (2, slots, "slots")], []
        for place, name, out in ((3, "k_stored", k_stored), (4, "v_stored", v_stored)):
            if out is not None:
                outs.append((place, contiguous(shaped(operand(out, name, (k.dtype,), 3, d), name, k.shape), name), name))
        held = [(5 + i, part, "the cache") for i, part in enumerate(self.arrays)]
        checks = overlaps(outs, ins)
        for part in held:
            checks += overlaps([part], ins + outs)
        return Plan("emmy_ops_cache4_append", a, self._FIELDS, checks)
