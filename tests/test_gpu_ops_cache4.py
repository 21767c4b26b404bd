"""The 4-bit cache on the B200: what it holds against the definition, bit for bit."""

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def stream():
    return torch.cuda.current_stream().cuda_stream


def cache(pages, heads, page, dim, fill=0):
    from emmyrt.cache4 import Cache4
    k, v = (torch.full((pages, heads, page, dim // 2), fill, dtype=torch.uint8, device="cuda") for _ in range(2))
    km, vm = (torch.full((pages, heads, page, 2), float(fill), dtype=torch.float16, device="cuda") for _ in range(2))
    return Cache4(k, km, v, vm), dict(k=k, v=v, k_meta=km, v_meta=vm)


def quantised(x):
    """levels, step, least of [.., dim] in the operator's own steps: f32 differences and a true division."""
    v = x.float().clamp(-65504, 65504)
    low, high = v.amin(-1, keepdim=True), v.amax(-1, keepdim=True)
    least = low.half()
    step = ((high - low).double() / 15).float().half()          # the f32 quotient, as f64 rounds it once more at most on ties
    s = step.float()
    n = torch.where(s > 0, ((v - least.float()).double() / s.double().clamp(min=1e-30)).float().round(), torch.zeros_like(v))
    return n.clamp(0, 15), step, least


def read(a, name, slot, page):
    bits, meta = a[name][slot // page, :, slot % page], a[name + "_meta"][slot // page, :, slot % page]
    return torch.stack((bits & 15, bits >> 4), -1).flatten(-2).float(), meta[..., :1], meta[..., 1:]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tokens,heads,page", [(1, 1, 1), (1, 8, 64), (5, 3, 7), (300, 2, 16)])
def test_append(runtime, dtype, dim, tokens, heads, page):
    g = torch.Generator(device="cuda").manual_seed(tokens)
    pages = -(-2 * tokens // page) + 1
    c, a = cache(pages, heads, page, dim, fill=7)
    k = (3 * torch.randn(tokens, heads, dim, generator=g, device="cuda")).to(TYPES[dtype])
    v = (0.1 * torch.randn(tokens, heads, dim, generator=g, device="cuda") + 5).to(TYPES[dtype])
    if tokens > 1:
        k[1] = 2.5                                              # all equal: step 0
        v[1] = 0
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens]
    ks, vs = torch.empty_like(k), torch.empty_like(v)
    c.append(k, v, slots.to(torch.int32) if dim == 64 else slots, k_stored=ks, v_stored=vs, stream=stream())
    for name, x, stored in (("k", k, ks), ("v", v, vs)):
        n, step, least = read(a, name, slots, page)
        rn, rs, rl = quantised(x)
        assert torch.equal(step, rs) and torch.equal(least, rl)
        assert torch.equal(n, rn)
        assert torch.equal(stored, (n * step.float() + least.float()).to(TYPES[dtype]))
    untouched = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    untouched[slots] = False
    rest = untouched.nonzero().flatten()
    for name in ("k", "v"):
        assert (a[name][rest // page, :, rest % page] == 7).all() and (a[name + "_meta"][rest // page, :, rest % page] == 7).all()


def test_slots_outside_are_left_out(runtime):
    c, a = cache(2, 1, 4, 64)
    k = torch.randn(6, 1, 64, device="cuda")
    out = torch.empty_like(k)
    c.append(k, k, torch.tensor([-1, 8, 3, 1 << 40, -(1 << 40), 7], device="cuda"), k_stored=out, stream=stream())
    held = [s for s in range(8) if (a["k_meta"][s // 4, 0, s % 4] != 0).any()]
    assert held == [3, 7] and (out.isfinite()).all()
    c.append(k[:0], k[:0], torch.zeros(0, dtype=torch.int64, device="cuda"), stream=stream())


def test_strides_and_extremes(runtime):
    """Keys and values inside a projection's rows, at any element; values past f16's range saturate, NaN stays NaN."""
    for shift in (0, 1):
        c, a = cache(1, 2, 8, 64)
        rows = torch.randn(4, 300, device="cuda").to(torch.bfloat16)
        k, v = (rows[:, o + shift:o + shift + 128].unflatten(1, (2, 64)) for o in (0, 128))
        k[0, 0, 3], k[1, 1, 0], v[2, 0, 9] = 3e38, float("-inf"), float("nan")
        slots = torch.arange(4, device="cuda")
        c.append(k, v, slots, stream=stream())
        n, step, least = read(a, "k", slots, 8)
        rn, rs, rl = quantised(k)
        assert torch.equal(n, rn) and torch.equal(step, rs) and torch.equal(least, rl)
        assert least[1, 1].item() == -65504
        n, step, least = read(a, "v", slots, 8)
        assert step[2, 0].isnan() and step.isnan().sum() == 1


def test_allocate(runtime):
    import numpy as np
    from emmyrt.cache4 import Cache4
    c = Cache4.allocate(3, 2, 5, 128)
    k = torch.randn(2, 2, 128, device="cuda")
    c.append(k, k, torch.tensor([0, 14], device="cuda"), stream=stream())
    torch.cuda.synchronize()
    held = c.k_meta.owner.download(np.zeros((3, 2, 5, 2), np.float16))
    assert (held[0, :, 0, 0] > 0).all() and (held[2, :, 4, 0] > 0).all() and (held != 0).sum() == 8


def test_append_right_after_allocate(runtime):
    """The zeros of a new cache are there before a stream that does not wait for the default one appends to it."""
    import numpy as np
    from emmyrt.cache4 import Cache4
    pages, heads, page, dim = 20000, 8, 64, 128            # 1.4 GB: its zeros take longer than a call
    k = torch.randn(2, heads, dim, device="cuda")
    slots = torch.tensor([0, pages * page - 1], device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    c = Cache4.allocate(pages, heads, page, dim)
    c.append(k, k, slots, stream=side.cuda_stream)
    torch.cuda.synchronize()
    for part in (c.k_meta, c.v_meta):
        held = part.owner.download(np.zeros((pages, heads, page, 2), np.float16))
        assert (held[0, :, 0, 0] > 0).all() and (held[-1, :, -1, 0] > 0).all() and (held != 0).sum() == 4 * heads
