"""What the operators' Python side refuses before anything is enqueued, on the CPU: operands are made-up addresses, and the
library's entries are replaced by one that records its call."""

import ctypes

import pytest


class Tensor:
    """Looks like a torch tensor."""

    class Device:
        def __init__(self, type, index):
            self.type, self.index = type, index

        def __eq__(self, other):
            return (self.type, self.index) == (other.type, other.index)

        def __hash__(self):
            return hash((self.type, self.index))

    def __init__(self, at, dtype, shape, strides, device=("cuda", 0)):
        self.at, self.dtype, self.shape, self.strides, self.device = at, dtype, shape, strides, Tensor.Device(*device)

    def data_ptr(self):
        return self.at

    def stride(self):
        return self.strides


@pytest.fixture
def calls(monkeypatch):
    """The operators on GPU 0, whose entries record (name, argument block)."""
    import emmyrt
    import emmyrt.blockfp8
    import emmyrt.cache4
    import emmyrt.operands
    import emmyrt.rotary
    made = []

    class Buffer:
        def __init__(self, nbytes):
            self.nbytes, self.ptr = nbytes, 1 << 50

        def upload(self, array):
            pass

        zero = upload

    kinds = {"emmy_ops_residual_norm": emmyrt.NormArgs, "emmy_ops_rotary": emmyrt.RotaryArgs,
             "emmy_ops_cache4_append": emmyrt.Cache4AppendArgs, "emmy_ops_cache4_attend": emmyrt.Cache4AttendArgs,
             "emmy_ops_blockfp8_quantize": emmyrt.BlockFp8QuantizeArgs, "emmy_ops_blockfp8_linear": emmyrt.BlockFp8LinearArgs}

    class Lib:
        def __init__(self):
            for name, kind in kinds.items():
                def entry(args, device, stream, name=name, kind=kind):
                    made.append((name, kind.from_buffer_copy(ctypes.string_at(args, ctypes.sizeof(kind)))))
                    return 0
                setattr(self, name, ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.c_int, ctypes.c_uint64)(entry))

        def emmy_ops_cache4_attend_workspace(self, dim, device, need):
            need._obj.value = 1 << 20
            return 0

    library = Lib()
    for module in (emmyrt.blockfp8, emmyrt.cache4, emmyrt.rotary):
        monkeypatch.setattr(module, "DeviceBuffer", Buffer)
    monkeypatch.setattr(emmyrt.operands, "current_device", lambda: 0)
    monkeypatch.setattr(emmyrt.operands, "ops_lib", lambda: library)
    monkeypatch.setattr(emmyrt.cache4, "ops_lib", lambda: library)
    monkeypatch.setattr(emmyrt.blockfp8.BlockFp8Linear, "_clear_status", lambda self: None)
    return made


def A(at, dtype, *shape, strides=None):
    from emmyrt.operands import Array
    return Array(at << 24, dtype, shape, strides)


def refuses(call, what):
    with pytest.raises(ValueError, match=what):
        call()


def test_arrays():
    from emmyrt.operands import Array, span
    assert Array(64, "f16", (3, 4)).strides == (4, 1)
    assert span(Array(64, "f16", (3, 4))) == 24 and span(Array(64, "f32", (2, 3), (10, 1))) == 52 and span(Array(64, "f32", (0, 3))) == 0

    class Owner:
        ptr, nbytes = 256, 24
    assert Array(Owner(), "f16", (3, 4)).ptr == 256
    refuses(lambda: Array(Owner(), "f16", (3, 5)), "in a buffer")
    refuses(lambda: Array(0, "f8", (3,)), "element type")
    refuses(lambda: Array(0, "f16", (-1,)), "shape")
    refuses(lambda: Array(0, "f16", (3, 4), (1,)), "strides")


def test_norm(calls):
    from emmyrt.norms import ResidualNorm
    for bad, what in ((dict(kind="group"), "kind"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps")):
        refuses(lambda: ResidualNorm(64, **bad), what)
    refuses(lambda: ResidualNorm(0), "dim")
    refuses(lambda: ResidualNorm(16385), "dim")
    op = ResidualNorm(64)
    x, b, y, h = (A(i, "bf16", 5, 64) for i in (1, 2, 3, 4))
    op(x, b, y, h)
    op(x, b, x, b)
    op(x, b, b, x)
    assert [n for n, _ in calls] == ["emmy_ops_residual_norm"] * 3 and calls[0][1].y == 3 << 24 and calls[1][1].y == 1 << 24
    w = A(5, "f32", 64)
    refuses(lambda: op(x, b, y, y), "overlaps")
    refuses(lambda: op(x, b, A(3, "f16", 5, 64)), "element type")
    refuses(lambda: op(x, b, A(3, "bf16", 4, 64)), "shape")
    refuses(lambda: op(A(1, "bf16", 5, 65), b, y), "columns")
    refuses(lambda: op(A(1, "bf16", 5, 64, strides=(1, 5)), b, y), "contiguous")
    refuses(lambda: op(x, b, A(3, "bf16", 5, 64, strides=(32, 1))), "overlap")
    refuses(lambda: op(x, b, y, pre_weight=w), "not asked for")
    refuses(lambda: ResidualNorm(64, post_norm=False)(x, b, y, post_weight=w), "post_norm")
    refuses(lambda: op(x, b, y, post_weight=A(5, "f32", 63)), "shape")
    refuses(lambda: op(x, b, y, post_weight=A(5, "e4m3", 64)), "element type")
    refuses(lambda: op(x, b, y, gate=A(5, "f32", 2, 64), rows_per_gate=2), "gate of shape")
    refuses(lambda: op(x, b, y, gate=A(5, "f32", 2, 64), rows_per_gate=0), "rows_per_gate")
    refuses(lambda: op(x, b, y, gate=A(3, "bf16", 1, 64)), "overlaps")
    refuses(lambda: op(x, b, "y"), "tensor is wanted")
    assert len(calls) == 3


def test_tensors_of_other_devices(calls):
    from emmyrt.norms import ResidualNorm
    op = ResidualNorm(8)
    make = lambda at, dtype="torch.float32", **kw: Tensor(at << 20, dtype, (2, 8), (8, 1), **kw)  # noqa: E731
    op(make(1), make(2), make(3))
    op(make(4), make(5), make(6))               # a call of a known kind
    assert len(calls) == 2 and calls[1][1].x == 4 << 20
    refuses(lambda: op(make(1), make(2), make(3, device=("cuda", 1))), "GPU 1")
    refuses(lambda: op(make(1), make(2), make(3, device=("cpu", None))), "not on a GPU")
    refuses(lambda: op(make(1), make(2), make(3, dtype="torch.float64")), "element type")
    refuses(lambda: op(make(1), make(2), Tensor((1 << 20) + 4, "torch.float32", (2, 8), (8, 1))), "overlaps")
    assert len(calls) == 2


def test_rotary(calls):
    import numpy as np
    from emmyrt.rotary import Rotary, frequencies
    for bad, what in ((dict(layout="pairs"), "layout"), (dict(scaling="dynamic"), "scaling"), (dict(rotary_dim=66), "rotary_dim"),
                      (dict(rotary_dim=7), "even"), (dict(rotary_dim=0), "rotary_dim"), (dict(base=0.0), "base"), (dict(factor=-1.0), "factor"),
                      (dict(scaling="parts", original_length=0), "original_length"), (dict(scaling="parts", slow=3, fast=3), "slow"),
                      (dict(rotary_dim=2, scaling="base", factor=2.0), "single pair"), (dict(magnitude=float("inf")), "magnitude")):
        refuses(lambda: Rotary(64, **bad), what)
    assert np.allclose(frequencies(4, 100.0), [1.0, 0.1]) and np.allclose(frequencies(4, 100.0, "linear", 2.0), [0.5, 0.05])
    f = frequencies(64, 10000.0, "base", 8.0)
    assert f[0] == 1.0 and np.isclose(f[-1], 10000.0 ** (-62 / 64) / 8)
    f, g = frequencies(64, 10000.0, "parts", 8.0, 4096), frequencies(64)
    assert np.array_equal(f[:2], g[:2]) and np.isclose(f[-1], g[-1] / 8)
    op = Rotary(64, 32)
    pos, q, k = A(1, "i32", 5), A(2, "bf16", 5, 4, 64), A(3, "bf16", 5, 1, 64)
    op(pos, q, k)
    op(pos, q, q_out=A(4, "bf16", 5, 4, 64), inverse=True)
    assert calls[0][1].out1 == 3 << 24 and calls[1][1].heads1 == 0 and calls[1][1].transpose == 1 and calls[0][1].transpose == 0
    refuses(lambda: op(A(1, "f32", 5), q), "element type")
    refuses(lambda: op(A(1, "i32", 6), q), "wanted")
    refuses(lambda: op(pos, A(2, "bf16", 5, 4, 32)), "wanted")
    refuses(lambda: op(pos, q, A(3, "f16", 5, 1, 64)), "element type")
    refuses(lambda: op(pos, q, k_out=k), "without k")
    refuses(lambda: op(pos, q, k, q_out=k), "shape")
    refuses(lambda: op(pos, q, A(2, "bf16", 5, 4, 64)), "overlaps")
    refuses(lambda: op(pos, A(2, "bf16", 5, 4, 64, strides=(0, 64, 1))), "overlap")
    rows = 24 << 20
    inside = lambda first, heads: A(0, "bf16", 5, heads, 64, strides=(384, 64, 1)).__class__(rows + 128 * first, "bf16", (5, heads, 64), (384, 64, 1))  # noqa: E731
    op(pos, inside(0, 4), inside(4, 2))         # side by side in one projection's rows
    refuses(lambda: op(pos, inside(0, 4), inside(3, 2)), "overlaps")
    assert len(calls) == 3


def cache_parts(pages=6, heads=2, page=16, dim=64):
    return (A(1, "u8", pages, heads, page, dim // 2), A(2, "f16", pages, heads, page, 2), A(3, "u8", pages, heads, page, dim // 2),
            A(4, "f16", pages, heads, page, 2))


def test_cache(calls):
    from emmyrt.cache4 import Cache4, Cache4Attention
    k, km, v, vm = cache_parts()
    refuses(lambda: Cache4(*cache_parts(dim=96)), "head dim")
    refuses(lambda: Cache4(k, km, k, vm), "overlaps")
    refuses(lambda: Cache4(k, A(2, "f16", 6, 2, 16, 3), v, vm), "shape")
    refuses(lambda: Cache4(k, km, A(3, "u8", 6, 2, 16, 32, strides=(2048, 1024, 32, 1)), vm), "contiguous")
    c = Cache4(k, km, v, vm)
    x, y, slots = A(5, "bf16", 3, 2, 64), A(6, "bf16", 3, 2, 64), A(7, "i64", 3)
    c.append(x, y, slots)
    c.append(x, x, slots, k_stored=A(8, "bf16", 3, 2, 64))
    assert calls[0][1].cache_pages == 6 and calls[0][1].slots_64 == 1 and calls[1][1].v_stored == 0
    refuses(lambda: c.append(x, y, A(7, "f32", 3)), "element type")
    refuses(lambda: c.append(x, y, A(7, "i64", 4)), "shape")
    refuses(lambda: c.append(A(5, "bf16", 3, 1, 64), y, slots), "shape")
    refuses(lambda: c.append(x, y, slots, k_stored=x), "overlaps")
    refuses(lambda: c.append(x, y, slots, k_stored=A(8, "f32", 3, 2, 64)), "element type")
    refuses(lambda: c.append(A(3, "bf16", 3, 2, 64), y, slots), "overlaps")
    refuses(lambda: Cache4Attention(c, 3), "heads")
    op = Cache4Attention(c, 8)
    q, out, table, lengths = A(9, "f16", 4, 1, 8, 64), A(10, "f16", 4, 1, 8, 64), A(11, "i32", 4, 3), A(12, "i32", 4)
    op(q, out, table, lengths)
    op(q, q, table, lengths, scale=0.0)
    assert calls[2][1].scale == 0.125 and calls[3][1].scale == 0.0 and calls[2][1].max_pages == 3
    refuses(lambda: op(A(9, "f32", 4, 1, 8, 64), out, table, lengths), "element type")
    refuses(lambda: op(A(9, "f16", 4, 1, 4, 64), out, table, lengths), "shape")
    refuses(lambda: op(q, out, A(11, "i64", 4, 3), lengths), "element type")
    refuses(lambda: op(q, out, A(11, "i32", 5, 3), lengths), "rows")
    refuses(lambda: op(q, out, table, A(12, "i32", 5)), "shape")
    refuses(lambda: op(q, A(2, "f16", 4, 1, 8, 64), table, lengths), "overlaps")
    refuses(lambda: op(q, out, table, lengths, scale=float("nan")), "scale")
    assert len(calls) == 4


def test_blockfp8(calls):
    from emmyrt.blockfp8 import BlockFp8Linear, BlockFp8Quantizer
    quantise = BlockFp8Quantizer()
    x, q, s = A(1, "f16", 6, 200), A(2, "u8", 6, 200, strides=(208, 1)), A(3, "f32", 2, 6)
    quantise(x, q, s)
    BlockFp8Quantizer(square=True)(x, q, A(3, "f32", 1, 2))
    refuses(lambda: quantise(x, A(2, "u8", 6, 200), s), "16")
    refuses(lambda: quantise(x, q, A(3, "f32", 6, 2)), "shape")
    refuses(lambda: quantise(A(1, "f16", 6, 0), A(2, "u8", 6, 0), s), "columns")
    refuses(lambda: quantise(A(2, "f16", 6, 200), q, s), "overlaps")
    wq, ws = A(4, "e4m3", 300, 200, strides=(208, 1)), A(5, "f32", 3, 2)
    refuses(lambda: BlockFp8Linear(A(4, "e4m3", 300, 200), ws, 8), "16")
    refuses(lambda: BlockFp8Linear(A(4, "f16", 300, 208), ws, 8), "element type")
    refuses(lambda: BlockFp8Linear(wq, A(5, "f32", 2, 2), 8), "shape")
    refuses(lambda: BlockFp8Linear(wq, ws, 0), "max_rows")
    op = BlockFp8Linear(wq, ws, 8)
    y = A(6, "bf16", 6, 300)
    op(x, y)
    assert calls[2][0] == "emmy_ops_blockfp8_linear" and calls[2][1].m == 6 and calls[2][1].xs_stride == 8
    refuses(lambda: op(A(1, "f16", 9, 200), A(6, "bf16", 9, 300)), "made for")
    refuses(lambda: op(A(1, "f16", 6, 208), y), "columns")
    refuses(lambda: op(x, A(6, "bf16", 6, 301)), "shape")
    refuses(lambda: op(x, A(5, "bf16", 6, 300)), "overlaps")
    refuses(lambda: op(x, A(6, "e4m3", 6, 300)), "element type")
    assert len(calls) == 3


def test_many_kinds_of_calls_are_not_kept_for_good(calls):
    from emmyrt.norms import ResidualNorm
    op = ResidualNorm(8)
    for rows in range(1, 2 * op.PLANS):
        op(A(1, "f32", rows, 8), A(2, "f32", rows, 8), A(3, "f32", rows, 8))
    assert len(op._plans) <= op.PLANS and calls[-1][1].rows == 2 * op.PLANS - 1


def test_allocate_waits_for_its_zeros(calls, monkeypatch):
    """The cache is all zero when allocate returns: streams that do not wait for the default stream, where it is zeroed, may append at once."""
    import emmyrt.cache4
    order = []

    class Buffer:
        def __init__(self, nbytes):
            self.nbytes, self.ptr = nbytes, (1 + len(order)) << 30

        def zero(self, stream=0):
            order.append(("zero", self.nbytes, stream))

    class Lib:
        def emmy_rt_stream_synchronize(self, stream):
            order.append(("wait", stream))
            return 0

    monkeypatch.setattr(emmyrt.cache4, "DeviceBuffer", Buffer)
    monkeypatch.setattr(emmyrt.cache4, "lib", Lib(), raising=False)
    emmyrt.cache4.Cache4.allocate(3, 2, 16, 64)
    assert order[:-1] == [("zero", 3 * 2 * 16 * 32, 0), ("zero", 3 * 2 * 16 * 4, 0)] * 2 and order[-1] == ("wait", 0)


@pytest.mark.parametrize("stream", [0, 77])
def test_from_weight_waits_for_its_weight(calls, monkeypatch, stream):
    """The quantised weight is there when from_weight returns, whatever stream it was quantised on and whatever stream calls come on."""
    import emmyrt.blockfp8
    order = []

    class Lib:
        def emmy_rt_stream_synchronize(self, s):
            order.append((s, len(calls)))
            return 0

    class Buffer:
        made = 0

        def __init__(self, nbytes):
            Buffer.made += 1
            self.nbytes, self.ptr = nbytes, Buffer.made << 40

    monkeypatch.setattr(emmyrt.blockfp8, "DeviceBuffer", Buffer)
    monkeypatch.setattr(emmyrt.blockfp8, "lib", Lib())
    op = emmyrt.blockfp8.BlockFp8Linear.from_weight(A(1, "bf16", 300, 200), 4, stream=stream)
    assert [n for n, _ in calls] == ["emmy_ops_blockfp8_quantize"] and calls[0][1].square == 1
    assert (stream, 1) in order and (op.n, op.k) == (300, 200)


def test_padding_stays_in_q(calls):
    """The row quantiser's zeros behind a row's last column: not where a single row has no room for them, and not past q's memory."""
    from emmyrt.blockfp8 import BlockFp8Quantizer
    from emmyrt.operands import Array

    class Owner:
        def __init__(self, nbytes):
            self.ptr, self.nbytes = 1 << 40, nbytes

    class Storage:
        def __init__(self, nbytes):
            self.size = nbytes

        def nbytes(self):
            return self.size

    class Held(Tensor):
        def __init__(self, nbytes, offset, *args):
            super().__init__(*args)
            self.memory, self.offset = Storage(nbytes), offset

        def untyped_storage(self):
            return self.memory

        def storage_offset(self):
            return self.offset

    quantise = BlockFp8Quantizer()
    x1, s1 = A(1, "f16", 1, 100), A(3, "f32", 1, 1)
    for q in (A(2, "u8", 1, 100), Array(Owner(100), "u8", (1, 100)), Tensor(2 << 24, "torch.uint8", (1, 100), (100, 1)),
              Tensor(2 << 24, "torch.uint8", (1, 100), (200, 1)), Tensor(2 << 24, "torch.uint8", (1, 100), (1, 1))):
        quantise(x1, q, s1)
        assert calls[-1][1].q_stride == 100             # of one row: no room for padding
    quantise(x1, A(2, "u8", 1, 100, strides=(128, 1)), s1)
    assert calls[-1][1].q_stride == 128
    quantise(x1, A(2, "u8", 1, 100), Array((2 << 24) + 100, "f32", (1, 1)))    # right behind such a row
    x, s = A(1, "f16", 3, 100), A(3, "f32", 1, 3)
    quantise(x, Array(Owner(2 * 112 + 112), "u8", (3, 100), (112, 1)), s)
    quantise(x, Held(500, 500 - 336, 2 << 24, "torch.uint8", (3, 100), (112, 1)), s)
    made = len(calls)
    refuses(lambda: quantise(x, Array(Owner(2 * 112 + 100), "u8", (3, 100), (112, 1)), s), "padding")
    refuses(lambda: quantise(x, Array(Owner(2 * 112 + 111), "u8", (3, 100), (112, 1)), s), "padding")
    refuses(lambda: quantise(x, Held(500, 500 - 335, 2 << 24, "torch.uint8", (3, 100), (112, 1)), s), "padding")
    refuses(lambda: quantise(x1, Array(Owner(100), "u8", (1, 100), (112, 1)), s1), "padding")
    assert len(calls) == made
    BlockFp8Quantizer(square=True)(x, Array(Owner(2 * 112 + 100), "u8", (3, 100), (112, 1)), A(3, "f32", 1, 1))


@pytest.mark.parametrize("current", [0, 1])
def test_status_waits_for_the_calls(calls, monkeypatch, current):
    """The status word is read when the calls before it are done: of all streams of the operator's device, or on the stream that is named,
    whichever device is current; a word that is set is cleared in the same order."""
    import emmyrt
    import emmyrt.blockfp8
    order, words = [], []

    class Lib:
        def emmy_rt_set_device(self, device):
            order.append(("device", device))
            return 0

        def emmy_rt_synchronize(self):
            order.append("all")
            return 0

        def emmy_rt_stream_synchronize(self, stream):
            order.append(("wait", stream))
            return 0

        def emmy_rt_memcpy_dtoh(self, to, at, nbytes, stream):
            order.append(("read", nbytes, stream))
            ctypes.c_uint32.from_address(to).value = words.pop(0)
            return 0

        def emmy_rt_memset(self, at, value, nbytes, stream):
            order.append(("clear", value, nbytes, stream))
            return 0

    op = emmyrt.blockfp8.BlockFp8Linear(A(4, "e4m3", 300, 208), A(5, "f32", 3, 2), 8)
    monkeypatch.setattr(emmyrt.blockfp8, "lib", Lib())
    monkeypatch.setattr(emmyrt.blockfp8, "current_device", lambda: current, raising=False)
    there, back = [("device", 0)], [("device", 1)] if current else []
    words += [0, 5, 0, 6]
    assert op.status() == 0 and order == there + ["all", ("read", 4, 0), ("wait", 0)] + back
    order.clear()
    assert op.status() == 5 and order == there + ["all", ("read", 4, 0), ("wait", 0), ("clear", 0, 4, 0), ("wait", 0)] + back
    order.clear()
    assert op.status(stream=77) == 0 and order == there + [("read", 4, 77), ("wait", 77)] + back
    order.clear()
    assert op.status(stream=77) == 6 and order == there + [("read", 4, 77), ("wait", 77), ("clear", 0, 4, 77), ("wait", 77)] + back


def test_numbers_that_f32_does_not_hold(calls):
    """Scales travel in f32: one that would become infinite there is refused, not rounded to infinity."""
    from emmyrt.cache4 import Cache4, Cache4Attention
    from emmyrt.norms import ResidualNorm
    from emmyrt.rotary import Rotary
    op = Cache4Attention(Cache4(*cache_parts()), 8)
    q, out, table, lengths = A(9, "f16", 4, 1, 8, 64), A(10, "f16", 4, 1, 8, 64), A(11, "i32", 4, 3), A(12, "i32", 4)
    for scale in (1e39, -1e300, float("inf"), 3e38):        # 3e38 is none in powers of two
        refuses(lambda: op(q, out, table, lengths, scale=scale), "scale")
    op(q, out, table, lengths, scale=2e38)
    for bad in (1e39, float("inf"), float("nan")):
        refuses(lambda: ResidualNorm(64, scale=bad), "scale")
        refuses(lambda: ResidualNorm(64, eps=bad), "eps")
        refuses(lambda: Rotary(64, magnitude=bad), "magnitude")
    ResidualNorm(64, scale=-3e38, eps=0.0)
    assert len(calls) == 1
