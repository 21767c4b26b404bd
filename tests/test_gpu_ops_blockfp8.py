"""FP8 products with a scale for each block of 128, on the B200.

The quantisers are checked bit for bit.  A product is checked against f64 sums of the same quantised values.  Its
tolerance: half a step of y's type; a block's 128 products are summed on the tensor cores, whose f32 sums may drop bits
below 2^-22 of the largest term at each of 4 steps of 32 (bounded here by 8 of 2^-22 of the sum of the products'
magnitudes), and the blocks' sums are added in f32: (blocks + 2) of 2^-24.
"""

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
E4M3 = torch.float8_e4m3fn


def stream():
    return torch.cuda.current_stream().cuda_stream


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def quantised(x, square):
    """(q as f32, s) in the operator's own steps"""
    rows, cols = x.shape
    rb, cb = -(-rows // 128), -(-cols // 128)
    p = torch.zeros(rb * 128 if square else rows, cb * 128, device="cuda")
    p[:rows, :cols] = x.float()
    b = p.view(rb, 128, cb, 128).transpose(1, 2) if square else p.view(rows, cb, 128)
    amax = b.abs().amax((2, 3) if square else 2)
    s = (amax.double() / 448).float()        # one rounding of the quotient, as the f32 division
    s = torch.where(s == 0, torch.ones_like(s), s)
    q = (b.double() / s.double()[..., None, None] if square else b.double() / s.double()[..., None]).float().to(E4M3).float()
    q = q.transpose(1, 2).reshape(rb * 128, cb * 128) if square else q.view(rows, cb * 128)
    return q[:rows, :cols], s if square else s.t()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("square", [False, True])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 130), (128, 128), (129, 257), (300, 1000), (5, 4096)])
def test_quantise(runtime, dtype, square, rows, cols):
    from emmyrt.blockfp8 import BlockFp8Quantizer, pitch
    x = torch.randn(rows, cols, generator=gen(rows), device="cuda") * 3
    x[:, 0] *= 100
    if cols > 128:
        x[:, 128:] = 0                       # blocks of zeros: scale 1
    x = x.to(TYPES[dtype])
    q = torch.full((rows, pitch(cols) + 16), 0x55, dtype=torch.uint8, device="cuda")
    s = torch.empty((-(-rows // 128), -(-cols // 128)) if square else (-(-cols // 128), rows), device="cuda")
    BlockFp8Quantizer(square)(x, q[:, :cols], s, stream=stream())
    rq, rs = quantised(x, square)
    assert torch.equal(s, rs)
    assert torch.equal(q[:, :cols].view(E4M3).float(), rq)
    assert (q[:, pitch(cols):] == 0x55).all()
    assert (q[:, cols:pitch(cols)] == (0x55 if square else 0)).all()


def test_quantise_strides_and_extremes(runtime):
    from emmyrt.blockfp8 import BlockFp8Quantizer
    for shift in (0, 1):
        wide = torch.randn(6, 300, device="cuda").to(torch.bfloat16)
        x = wide[:, shift:shift + 256]
        x[0, 3], x[1, 200], x[2, 5], x[3, 0] = float("nan"), float("inf"), 3e38, 0
        x[4] = 1e-40                         # subnormal: the scale is too
        q, s = torch.empty(6, 256, dtype=E4M3, device="cuda"), torch.empty(2, 6, device="cuda")
        BlockFp8Quantizer()(x, q, s, stream=stream())
        assert s[0, 0].isnan() and q[0, :128].float().isnan().all() and q[0, 128:].float().isfinite().all()
        assert s[1, 1].isinf() and q[1, 200].float().isnan() and (q[1, 128:200].float() == 0).all()
        fine = [2, 3, 5]
        rq, rs = quantised(x[fine], False)
        assert torch.equal(s[:, fine], rs) and torch.equal(q[fine].float(), rq)
        assert (s[:, 4] > 0).all() and (s[:, 4] < 1e-40).all()


def weights(n, k, seed=0):
    g = gen(seed)
    pitch = -(-k // 16) * 16
    wq = torch.full((n, pitch), float("nan"), device="cuda").to(E4M3)         # the padding is not to be read as numbers
    wq[:, :k] = (torch.randn(n, k, generator=g, device="cuda") * 60).clamp(-448, 448).to(E4M3)
    ws = (0.5 + torch.rand(-(-n // 128), -(-k // 128), generator=g, device="cuda")) * 0.01
    return wq[:, :k], ws


def reference(x, wq, ws, out):
    (m, k), n = x.shape, wq.shape[0]
    xq, xs = quantised(x, False)
    y = torch.zeros(m, n, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(y)
    rows = torch.arange(n, device="cuda") // 128
    for b in range(ws.shape[1]):
        c = slice(128 * b, min(k, 128 * b + 128))
        s = xs[b].double()[:, None] * ws[rows, b].double()
        u, v = xq[:, c].double(), wq[:, c].double()
        y += u @ v.t() * s
        size += u.abs() @ v.abs().t() * s
    return y, size * (8 * 2.0 ** -22 + (ws.shape[1] + 2) * 2.0 ** -24) + torch.finfo(out).eps / 2 * y.abs() + torch.finfo(out).tiny


def check(m, n, k, x_type="bf16", y_type="bf16", seed=0):
    from emmyrt.blockfp8 import BlockFp8Linear
    wq, ws = weights(n, k, seed)
    x = torch.randn(m, k, generator=gen(seed + 1), device="cuda")
    x[:, ::50] *= 20
    x = x.to(TYPES[x_type])
    y = torch.full((m, n), float("nan"), dtype=TYPES[y_type], device="cuda")
    op = BlockFp8Linear(wq, ws, max_rows=m + 3)
    op(x, y, stream=stream())
    ref, bound = reference(x, wq, ws, TYPES[y_type])
    worst = ((y.double() - ref).abs() - bound).max().item()
    assert worst <= 0, f"off by {worst} more than the bound"
    assert op.status() == 0
    return op, x, y


@pytest.mark.parametrize("m", [1, 2, 7, 8, 9, 16, 17, 32, 33, 64, 127, 128, 129, 200, 256, 300])
@pytest.mark.parametrize("n,k", [(1, 1), (8, 16), (128, 128), (100, 200), (272, 160), (513, 1040), (1024, 2000)])
def test_product(runtime, m, n, k):
    check(m, n, k, y_type="f32")


@pytest.mark.parametrize("m", [1, 2, 3, 8, 16])
@pytest.mark.parametrize("n,k", [(2400, 1500), (2368, 1025), (4101, 4200), (40, 12000), (9000, 1000)])
def test_few_rows(runtime, m, n, k):
    check(m, n, k)


@pytest.mark.parametrize("x_type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("y_type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m", [5, 150])
def test_types(runtime, x_type, y_type, m):
    check(m, 300, 700, x_type, y_type)


@pytest.mark.parametrize("m,n,k", [(1024, 4096, 512), (2048, 2048, 1024), (1000, 3001, 1500), (4097, 1300, 257), (129, 20000, 300),
                                   (257, 19000, 130)])
def test_large(runtime, m, n, k):
    """Sizes that take the widest tiles, on pairs of SMs, and more tiles than SMs."""
    check(m, n, k)


def test_strides_rows_and_repeats(runtime):
    """x and y inside wider rows, fewer rows than planned, the same bits again, rows behind the last one left as they are."""
    from emmyrt.blockfp8 import BlockFp8Linear
    wq, ws = weights(384, 640)
    op = BlockFp8Linear(wq, ws, max_rows=300)
    for m in (300, 3, 40, 200):
        for shift in (0, 3):
            xw = torch.randn(m, 700, device="cuda").half()
            yw = torch.full((m + 2, 400), 7.0, device="cuda", dtype=torch.bfloat16)
            x, y = xw[:, shift:shift + 640], yw[:m, shift:shift + 384]
            op(x, y, stream=stream())
            first = y.clone()
            op(x, y, stream=stream())
            assert torch.equal(first, y)
            ref, bound = reference(x, wq, ws, torch.bfloat16)
            assert ((y.double() - ref).abs() <= bound).all()
            assert (yw[m:] == 7).all() and (yw[:, :shift] == 7).all() and (yw[:, shift + 384:] == 7).all()
    op(torch.zeros(0, 640, device="cuda"), torch.zeros(0, 384, device="cuda"), stream=stream())


def test_not_finite_stays_in_its_row(runtime):
    from emmyrt.blockfp8 import BlockFp8Linear
    wq, ws = weights(256, 300)
    for m in (4, 140):
        x = torch.randn(m, 300, device="cuda")
        x[1, 299], x[2, 0] = float("nan"), float("inf")
        y = torch.empty(m, 256, device="cuda")
        BlockFp8Linear(wq, ws, max_rows=m)(x, y, stream=stream())
        assert y[1].isnan().all() and not y[2].isfinite().any()
        rest = [i for i in range(m) if i not in (1, 2)]
        assert y[rest].isfinite().all()


def test_from_weight(runtime):
    from emmyrt.blockfp8 import BlockFp8Linear
    w = torch.randn(200, 333, device="cuda").to(torch.bfloat16)
    x = torch.randn(50, 333, device="cuda").to(torch.bfloat16)
    y = torch.empty(50, 200, device="cuda")
    BlockFp8Linear.from_weight(w, 50, stream=stream())(x, y, stream=stream())
    wq, ws = quantised(w, True)
    ref, bound = reference(x, wq, ws, torch.float32)
    assert ((y.double() - ref).abs() <= bound).all()


def test_graph(runtime):
    op, x, y = check(70, 500, 600)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        op(x, y, stream=stream())
    for seed in (3, 4):
        x.copy_(torch.randn(70, 600, generator=gen(seed), device="cuda"))
        g.replay()
        torch.cuda.synchronize()
        again = torch.empty_like(y)
        op(x, again, stream=stream())
        assert torch.equal(again, y)


@pytest.mark.parametrize("x_type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,n,k", [(1, 40, 300), (2, 500, 1000), (2, 3000, 2600), (1, 1, 1), (1, 4096, 4096), (3, 40, 300), (40, 300, 700)])
def test_linear_leaves_the_quantised_x(runtime, x_type, m, n, k):
    """The C entry's contract: x stands quantised in xq and xs after the call, its padding zero, at sizes that quantise it within
    the product too, so that a second product can share it."""
    import ctypes
    import emmyrt
    wq, ws = weights(n, k)
    x = torch.randn(m, k, generator=gen(9), device="cuda").to(TYPES[x_type])
    x[0, 0] = 100
    pitch = -(-k // 16) * 16
    xq = torch.full((m, pitch + 16), 0x55, dtype=torch.uint8, device="cuda")
    xs = torch.full((-(-k // 128) + 1, -(-m // 4) * 4), -1.0, device="cuda")
    y, again = (torch.full((m, n), float("nan"), device="cuda") for _ in range(2))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    a = emmyrt.BlockFp8LinearArgs(xq=xq.data_ptr(), xs=xs.data_ptr(), wq=wq.data_ptr(), ws=ws.data_ptr(), y=y.data_ptr(),
                                  status=status.data_ptr(), xq_stride=pitch + 16, xs_stride=xs.stride(0), wq_stride=pitch,
                                  ws_stride=ws.stride(0), y_stride=n, m=m, n=n, k=k, dtype=0, x=x.data_ptr(), x_stride=k,
                                  x_dtype=["f32", "f16", "bf16"].index(x_type))
    assert emmyrt.ops_lib().emmy_ops_blockfp8_linear(ctypes.byref(a), 0, stream()) == 0
    rq, rs = quantised(x, False)
    assert torch.equal(xs[:-1, :m], rs) and (xs[-1] == -1).all() and (xs[:, m:] == -1).all()
    assert torch.equal(xq[:, :k].view(E4M3).float(), rq)
    assert (xq[:, k:pitch] == 0).all() and (xq[:, pitch:] == 0x55).all()
    # the product alone, of what the call left
    p = emmyrt.BlockFp8Args(**{f: getattr(a, f) for f, _ in emmyrt.BlockFp8Args._fields_})
    p.y = again.data_ptr()
    assert emmyrt.ops_lib().emmy_ops_blockfp8_product(ctypes.byref(p), 0, stream()) == 0
    ref, bound = reference(x, wq, ws, torch.float32)
    for out in (y, again):
        assert ((out.double() - ref).abs() <= bound).all()
    assert status.item() == 0


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cols", [1, 7, 8, 9, 15, 16, 17, 100, 130, 1025])
def test_quantise_a_row_without_padding(runtime, dtype, cols):
    """A single row in exactly its own bytes: what stands behind it stays."""
    from emmyrt.blockfp8 import BlockFp8Quantizer
    x = torch.randn(1, cols, generator=gen(cols), device="cuda").to(TYPES[dtype])
    held = torch.full((3, cols), 0x55, dtype=torch.uint8, device="cuda")
    s = torch.empty(-(-cols // 128), 1, device="cuda")
    BlockFp8Quantizer()(x, held[:1], s, stream=stream())
    rq, rs = quantised(x, False)
    assert torch.equal(s, rs) and torch.equal(held[:1].view(E4M3).float(), rq) and (held[1:] == 0x55).all()


def test_status_of_calls_on_other_streams(runtime):
    """status() waits for a call on a stream that the default one does not wait for: a word that is set behind it is seen, once."""
    from emmyrt.blockfp8 import BlockFp8Linear
    wq, ws = weights(2048, 2048)
    op = BlockFp8Linear(wq, ws, max_rows=4096)
    x, y = torch.randn(4096, 2048, device="cuda").half(), torch.empty(4096, 2048, device="cuda")
    word = torch.full((1,), 8, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for named in (None, side.cuda_stream):
        for _ in range(30):
            op(x, y, stream=side.cuda_stream)
        runtime.check(runtime.lib.emmy_rt_memcpy_dtod(op._status, word.data_ptr(), 4, side.cuda_stream), "copy")
        assert op.status(stream=named) == 8 and op.status(stream=named) == 0


@pytest.mark.parametrize("m", [2, 5, 40, 150])
def test_one_row_for_all(runtime, m):
    """x broadcast over its rows (stride 0): quantised and multiplied like the rows written out."""
    from emmyrt.blockfp8 import BlockFp8Linear, BlockFp8Quantizer
    wq, ws = weights(200, 330)
    x = torch.randn(1, 330, generator=gen(m), device="cuda").half().expand(m, 330)
    y, z = (torch.empty(m, 200, device="cuda") for _ in range(2))
    op = BlockFp8Linear(wq, ws, max_rows=m)
    op(x, y, stream=stream())
    op(x.contiguous(), z, stream=stream())
    assert torch.equal(y, z)
    for square in (False, True):
        got = []
        for v in (x, x.contiguous()):
            q = torch.zeros(m, 336, dtype=torch.uint8, device="cuda")
            s = torch.empty((-(-m // 128), 3) if square else (3, m), device="cuda")
            BlockFp8Quantizer(square)(v, q[:, :330], s, stream=stream())
            got.append((q, s))
        assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


def test_call_and_status_from_a_new_thread(runtime):
    """A thread that has used no device yet may call an operator and ask for its status."""
    import threading
    op, x, y = check(9, 300, 400)
    again = torch.empty_like(y)
    torch.cuda.synchronize()
    got = []
    on = stream()
    threads = [threading.Thread(target=lambda: got.append(op.status())),
               threading.Thread(target=lambda: (op(x, again, stream=on), got.append(op.status())))]
    for t in threads:
        t.start()
        t.join()
    assert got == [0, 0] and torch.equal(y, again)
