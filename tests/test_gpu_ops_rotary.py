"""Rotary positions on the B200 against cosines and sines in f64.

Tolerances: half a step of the type, and in f32 the angle (a turn's fraction to 2^-25 of a half turn: pi 2^-25
radians), cosine and sine (2 ulp), two products and a sum: 8 of 2^-24 of |a| + |b|, times the magnitude.
"""

import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def frequency(i, r, base, scaling, factor, original):
    if scaling == "base":
        base *= factor ** (r / (r - 2))
    f = base ** (-2 * i / r)
    if scaling == "linear":
        return f / factor
    if scaling == "parts":
        keep = min(1, max(0, (original * f / (2 * math.pi) - 1) / 31))
        return f * keep + f / factor * (1 - keep)
    return f


def reference(x, positions, r, layout, inverse, base=10000.0, scaling="none", factor=1.0, original=4096, magnitude=1.0):
    x = x.double()
    f = torch.tensor([frequency(i, r, base, scaling, factor, original) for i in range(r // 2)], dtype=torch.float64,
                     device=x.device)
    t = positions.double()[:, None, None] * f * (-1 if inverse else 1)
    c, s = t.cos() * magnitude, t.sin() * magnitude
    ia, ib = (range(r // 2), range(r // 2, r)) if layout == "half" else (range(0, r, 2), range(1, r, 2))
    a, b = x[..., list(ia)], x[..., list(ib)]
    out, bound = x.clone(), torch.zeros_like(x)
    out[..., list(ia)], out[..., list(ib)] = a * c - b * s, a * s + b * c
    bound[..., list(ia)] = bound[..., list(ib)] = 8 * 2.0 ** -24 * (a.abs() + b.abs()) * magnitude
    return out, bound


def close(got, x, positions, *args, **kw):
    ref, bound = reference(x, positions, *args, **kw)
    step = torch.finfo(got.dtype).eps / 2 * ref.abs() + torch.finfo(got.dtype).tiny
    worst = ((got.double() - ref).abs() - step - bound).max().item() if ref.numel() else 0
    assert worst <= 0, f"off by {worst} more than the bound"


def stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("tokens,heads,kv,dim,rotary", [(1, 1, 1, 2, 2), (1, 32, 8, 128, 128), (7, 5, 1, 64, 32), (3, 2, 2, 80, 20),
                                                        (2, 3, 1, 66, 66), (5, 1, 2, 96, 64), (700, 4, 4, 64, 16),
                                                        (2, 1, 1, 8192, 8192)])
def test_shapes(runtime, dtype, layout, inverse, tokens, heads, kv, dim, rotary):
    from emmyrt.rotary import Rotary
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(tokens, heads, dim, generator=g, device="cuda").to(TYPES[dtype])
    k = torch.randn(tokens, kv, dim, generator=g, device="cuda").to(TYPES[dtype])
    pos = torch.randint(0, 1 << 21, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    op = Rotary(dim, rotary, layout=layout)
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    op(pos, q, k, q_out=qo, k_out=ko, inverse=inverse, stream=stream())
    close(qo, q, pos, rotary, layout, inverse)
    close(ko, k, pos, rotary, layout, inverse)
    op(pos.long(), q, inverse=inverse, stream=stream())           # in place, int64, on its own
    assert torch.equal(q, qo)


@pytest.mark.parametrize("scaling,factor", [("linear", 8.0), ("base", 4.0), ("parts", 32.0), ("parts", 1.5)])
@pytest.mark.parametrize("rotary", [128, 48])
def test_scalings(runtime, scaling, factor, rotary):
    from emmyrt.rotary import Rotary
    q = torch.randn(50, 3, 128, device="cuda")
    pos = torch.arange(50, device="cuda") * 20011
    magnitude = 0.1 * math.log(factor) + 1 if scaling == "parts" else 1.0
    out = torch.empty_like(q)
    Rotary(128, rotary, base=5e5, scaling=scaling, factor=factor, original_length=8192)(pos, q, q_out=out, stream=stream())
    close(out, q, pos, rotary, "half", False, 5e5, scaling, factor, 8192, magnitude)


def test_positions_far_and_negative(runtime):
    """2^40 and below zero: the angle wraps in 64 bits.  A frequency of at most 1 is known to 2^-53 on either side, and the
    reference rounds its product, the operator its quotient by 2 pi and the fraction of 64 bits: the angles differ by less
    than 4 of 2^-53 of the position, and the result by that much of |a| + |b| (the bound's 8 of 2^-24)."""
    from emmyrt.rotary import Rotary
    q = torch.randn(6, 2, 64, device="cuda")
    pos = torch.tensor([0, -1, -77777, (1 << 31) - 1, 1 << 33, (1 << 40) + 3], device="cuda")
    out = torch.empty_like(q)
    Rotary(64)(pos, q, q_out=out, stream=stream())
    ref, bound = reference(q, pos, 64, "half", False)
    angle = 4 * 2.0 ** -53 * pos.abs().double()[:, None, None]
    worst = ((out.double() - ref).abs() - bound * (1 + angle / (8 * 2.0 ** -24)) - 2.0 ** -24 * ref.abs()).max().item()
    assert worst <= 0, f"off by {worst} more than the bound"
    assert torch.equal(out[0], q[0])


def test_strides(runtime):
    """Queries and keys inside one projection's rows, at offsets that 16-byte accesses cannot take."""
    from emmyrt.rotary import Rotary
    pos = torch.arange(9, device="cuda", dtype=torch.int32) * 100
    for shift in (0, 2, 3):
        rows = torch.randn(9, 4 * 64 + 8, device="cuda").to(torch.bfloat16)
        before = rows.clone()
        q = rows[:, shift:shift + 192].unflatten(1, (3, 64))
        k = rows[:, shift + 192:shift + 256].unflatten(1, (1, 64))
        for layout in ("half", "interleaved"):
            rows.copy_(before)
            Rotary(64, 32, layout=layout)(pos, q, k, stream=stream())
            close(rows[:, shift:shift + 256].unflatten(1, (4, 64)), before[:, shift:shift + 256].unflatten(1, (4, 64)), pos, 32, layout, False)
            assert torch.equal(rows[:, :shift], before[:, :shift]) and torch.equal(rows[:, shift + 256:], before[:, shift + 256:])


def test_gradient(runtime):
    """The transposed map is the gradient: <R x, g> = <x, R' g>, and differences of a loss agree with it.  The loss is linear
    in x, so a difference over any step is exact but for rounding."""
    from emmyrt.rotary import Rotary
    op = Rotary(32, 24, layout="interleaved", scaling="parts", factor=4.0)
    pos = torch.tensor([3, 1000, 70000], device="cuda")
    x, g = torch.randn(2, 3, 2, 32, device="cuda").unbind(0)
    grad, y = torch.empty_like(x), torch.empty_like(x)
    op(pos, g, q_out=grad, inverse=True, stream=stream())
    op(pos, x, q_out=y, stream=stream())
    for i, j, e in ((0, 0, 0), (1, 1, 7), (2, 0, 23), (2, 1, 30)):
        moved, ym = x.clone(), torch.empty_like(x)
        moved[i, j, e] += 1.0
        op(pos, moved, q_out=ym, stream=stream())
        slope = ((ym - y).double() * g.double()).sum().item()
        # y's differences: two roundings of values below 8 (2^-21), over the 2 elements they reach, times |g| below 5
        assert abs(slope - grad[i, j, e].item()) < 4 * 2.0 ** -21 * 5 + 64 * 2.0 ** -24


def test_no_tokens(runtime):
    from emmyrt.rotary import Rotary
    Rotary(64)(torch.zeros(0, device="cuda", dtype=torch.int32), torch.zeros(0, 4, 64, device="cuda"), stream=stream())
