"""Device arrays as the operators take them, and the checks that every call makes.

An operand is an :class:`Array` (a pointer with its element type, shape and strides, for instance
over a :class:`emmyrt.DeviceBuffer`) or any object with ``data_ptr()``, ``dtype``, ``shape``,
``stride()`` and ``device``, as a torch tensor has.  Checks raise ``ValueError`` before anything is
enqueued; a call that the library refuses raises :class:`emmyrt.EmmyRTError`.
"""

from __future__ import annotations

import ctypes
import math

from . import EmmyRTError, _calls, current_device, ops_lib

CODE = {"f32": 0, "f16": 1, "bf16": 2}
ITEMSIZE = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1, "u8": 1, "i32": 4, "i64": 8, "f64": 8, "u64": 8}
FLOATS = ("f32", "f16", "bf16")
INDICES = ("i32", "i64")

_NAMES = {"torch.float32": "f32", "torch.float16": "f16", "torch.bfloat16": "bf16", "torch.float8_e4m3fn": "e4m3",
          "torch.uint8": "u8", "torch.int32": "i32", "torch.int64": "i64"}
_seen: dict = {}            # dtype object -> name, as str(dtype) costs more than the rest of a check


def f32(value: float) -> bool:
    """Whether f32 holds a number of this size."""
    return math.isfinite(ctypes.c_float(value).value)


class Array:
    """``shape`` elements of ``dtype`` at ``at`` (an address, or an owner with ``ptr``), rows first
    unless ``strides`` (in elements) says otherwise."""

    __slots__ = ("ptr", "dtype", "shape", "strides", "device", "owner")

    def __init__(self, at, dtype: str, shape, strides=None, device: int | None = None):
        self.owner = at
        self.ptr = int(getattr(at, "ptr", at))
        if dtype not in ITEMSIZE:
            raise ValueError(f"element type {dtype!r} is not one of {', '.join(ITEMSIZE)}")
        self.dtype = dtype
        self.shape = tuple(int(n) for n in shape)
        if any(n < 0 for n in self.shape):
            raise ValueError(f"shape {self.shape}")
        if strides is None:
            strides, n = [], 1
            for extent in reversed(self.shape):
                strides.append(n)
                n *= extent
            strides.reverse()
        self.strides = tuple(int(n) for n in strides)
        if len(self.strides) != len(self.shape):
            raise ValueError(f"{len(self.strides)} strides for a shape of {len(self.shape)}")
        self.device = device
        held = getattr(at, "nbytes", None)
        if held is not None and span(self) > held:
            raise ValueError(f"{span(self)} bytes of {dtype} {self.shape} in a buffer of {held}")


_calls.set_array(Array)


def span(a: Array) -> int:
    """Bytes from the first element to the end of the last one."""
    if 0 in a.shape:
        return 0
    return (sum((n - 1) * s for n, s in zip(a.shape, a.strides)) + 1) * ITEMSIZE[a.dtype]


def row_span(a: Array) -> int:
    """Bytes from the first element to the end of the last one of a first-dimension row."""
    return (sum((n - 1) * s for n, s in zip(a.shape[1:], a.strides[1:])) + 1) * ITEMSIZE[a.dtype]


def operand(x, name: str, dtypes, ndim: int, device: int) -> Array:
    """``x`` as an Array of ``ndim`` dimensions whose last one is contiguous."""
    if type(x) is Array:
        a = x
    elif hasattr(x, "data_ptr"):
        dtype = _seen.get(x.dtype)
        if dtype is None:
            dtype = _NAMES.get(str(x.dtype))
            if dtype is None:
                raise ValueError(f"{name}: element type {x.dtype}")
            _seen[x.dtype] = dtype
        where = x.device
        if where.type != "cuda":
            raise ValueError(f"{name} is on {where}, not on a GPU")
        a = Array.__new__(Array)
        a.ptr, a.dtype, a.shape, a.strides, a.device, a.owner = x.data_ptr(), dtype, x.shape, x.stride(), where.index, x
    else:
        raise ValueError(f"{name}: an Array or a tensor is wanted, not {type(x).__name__}")
    if a.device is not None and a.device != device:
        raise ValueError(f"{name} is on GPU {a.device}, the operator on GPU {device}")
    if a.dtype not in dtypes:
        raise ValueError(f"{name}: element type {a.dtype}, wanted {' or '.join(dtypes)}")
    if len(a.shape) != ndim:
        raise ValueError(f"{name} has {len(a.shape)} dimensions, wanted {ndim}")
    if ndim and a.strides[-1] != 1 and a.shape[-1] > 1:
        raise ValueError(f"{name}: the last dimension is not contiguous")
    if any(s < 0 for s in a.strides):
        raise ValueError(f"{name}: negative stride")
    return a


def shaped(a: Array, name: str, shape) -> Array:
    if tuple(a.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(a.shape)}, wanted {tuple(shape)}")
    return a


def contiguous(a: Array, name: str) -> Array:
    n = 1
    for extent, stride in zip(reversed(a.shape), reversed(a.strides)):
        if extent > 1 and stride != n:
            raise ValueError(f"{name} is not contiguous")
        n *= extent
    return a


def written(a: Array, name: str) -> Array:
    """An operand that the call writes: no two of its elements may share memory."""
    reach = 1
    for stride, extent in sorted((s, n) for s, n in zip(a.strides, a.shape) if n > 1):
        if stride < reach:
            raise ValueError(f"{name}: elements overlap (strides {tuple(a.strides)})")
        reach = stride * (extent - 1) + reach
    return a


class Apart:
    """The check that an output does not overlap another operand, prepared for two places of a call."""

    __slots__ = ("i", "j", "span_i", "span_j", "same", "step", "row_i", "row_j", "name")

    def __init__(self, i: int, out: Array, j: int, other: Array, name: str, same: bool):
        self.i, self.j, self.span_i, self.span_j, self.name = i, j, span(out), span(other), name
        self.same = same and tuple(out.shape) == tuple(other.shape) and out.dtype == other.dtype and \
            all(p == q for p, q, n in zip(out.strides, other.strides, out.shape) if n > 1)
        # rows side by side in wider rows, as the parts of one projection are
        self.step = 0
        if self.span_i and self.span_j and out.shape and other.shape:
            step = out.strides[0] * ITEMSIZE[out.dtype]
            if step > 0 and step == other.strides[0] * ITEMSIZE[other.dtype]:
                self.step, self.row_i, self.row_j = step, row_span(out), row_span(other)

    def meets(self, p: int, q: int) -> None:
        """``p`` and ``q`` are the operands' addresses, whose spans overlap."""
        if self.same and p == q:
            return
        if self.step:
            gap = (q - p) % self.step
            if self.row_i <= gap and gap + self.row_j <= self.step:
                return
        raise ValueError(f"{self.name} overlaps another operand of the call")


def apart(out: Array, other: Array, name: str, *, same: bool) -> None:
    """``out`` must not overlap ``other``; with ``same`` it may be the very same elements."""
    check = Apart(0, out, 1, other, name, same)
    if out.ptr < other.ptr + check.span_j and other.ptr < out.ptr + check.span_i:
        check.meets(out.ptr, other.ptr)


def own_device() -> int:
    """The device an operator is made for: the one that is current."""
    return current_device()


def plan(name: str, args: ctypes.Structure, fields, checks, own=()) -> "_calls.Plan":
    """What calls with operands of the same types, shapes and strides have in common: the entry, the argument block without
    the operands' addresses (``fields`` names them, one for each operand) and the overlaps to look for.  ``own``: the
    operator's own arrays, whose places come after the operands'."""
    entry = ctypes.cast(getattr(ops_lib(), name), ctypes.c_void_p).value
    wanted = [(c.i, c.j, c.span_i, c.span_j, c.meets) for c in checks if c.span_i and c.span_j]
    return _calls.Plan(entry, bytes(args), tuple(getattr(type(args), f).offset for f in fields), tuple(a.ptr for a in own), wanted)


class Operator:
    """An operator of one device.  A call's operands are checked in full the first time that their types, shapes and
    strides come; later calls like it look only at the addresses.  Calls keep no state, so threads may share one."""

    PLANS = 512         # calls of so many kinds are remembered

    def __init__(self):
        self.device = own_device()
        self._plans: dict = {}

    def _plan(self, operands, options) -> tuple:
        """The arguments of :func:`plan` for a call, or a ``ValueError`` that says what is wrong with it."""
        raise NotImplementedError

    def _call(self, operands, options, stream: int) -> None:
        status = _calls.call(self._plans, operands, options, self.device, stream)
        while type(status) is not int:      # the call's kind, which the plans do not have (yet, or any more)
            what = self._plan(operands, options)
            if status is None:
                raise ValueError("an operand is neither an Array nor a tensor")
            if len(self._plans) >= self.PLANS:
                self._plans.clear()
            self._plans[status] = plan(*what)
            status = _calls.call(self._plans, operands, options, self.device, stream)
        if status:
            raise EmmyRTError(status, type(self).__name__, ops_lib().emmy_ops_last_error().decode(errors="replace"))


def overlaps(outs, others, *, same=()) -> list:
    """The checks of every output against the others and against each other: ``outs`` and ``others`` are
    (place, Array or None, name); ``same`` the pairs of places that may be the very same elements."""
    checks = []
    outs = [o for o in outs if o[1] is not None]
    for n, (i, out, name) in enumerate(outs):
        for j, other, _ in (*outs[:n], *others):
            if other is not None:
                checks.append(Apart(i, out, j, other, name, (i, j) in same))
    return checks
