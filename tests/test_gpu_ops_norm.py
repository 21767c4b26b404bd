"""The residual norm on the B200 against its definition in f64.

Tolerances: an output is off by half a step of its type, and by the f32 arithmetic.  A row's sum of
squares is added in chains of at most 16 and trees of at most 10 levels, so it is off by 26 of 2^-24
relative, its root by half of that; with the handful of products and sums after it every term of y is
off by less than 32 of 2^-24 of the terms' magnitudes.  h divides by the deviation of y, so y's error
enters relative to it: 64 of 2^-24 of |y| / deviation, times the weight.
"""

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24


def normalised(v, layer, eps, w, b):
    mean = v.mean(-1, keepdim=True) if layer else torch.zeros_like(v[:, :1])
    std = ((v - mean) ** 2).mean(-1, keepdim=True).add(eps).sqrt()
    out = (v - mean) / std
    if w is not None:
        out = out * w.double()
    return (out if b is None else out + b.double()), std


def reference(t, kind, eps, scale, post_norm, per):
    """(y, bound on its f32 error, h, bound) in f64; t: the operands by name."""
    x, n = t["x"].double(), t["block"].double()
    layer = kind == "layer"
    grow = torch.zeros_like(n)
    if post_norm:
        n, std = normalised(n, layer, eps, t.get("post_weight"), t.get("post_bias"))
        if layer:      # the mean is off relative to the largest value of the row
            grow = t["block"].double().abs().amax(-1, keepdim=True) / std
            if t.get("post_weight") is not None:
                grow = grow * t["post_weight"].double().abs()
    if t.get("gate") is not None:
        g = t["gate"].double()[torch.arange(x.shape[0], device=x.device) // per]
        n, grow = n * g, grow * g.abs()
    y = x + scale * n
    ty = 32 * U * (x.abs() + abs(scale) * (n.abs() + grow))
    h, std = normalised(y, layer, eps, t.get("pre_weight"), t.get("pre_bias"))
    w = t["pre_weight"].double().abs() if t.get("pre_weight") is not None else 1.0
    th = (64 * U * y.abs().amax(-1, keepdim=True) + 2 * ty.amax(-1, keepdim=True)) / std * w + 8 * U * h.abs()
    return y, ty, h, th


def close(got, ref, bound, dtype):
    step = torch.finfo(dtype).eps / 2 * ref.abs() + torch.finfo(dtype).tiny
    worst = ((got.double() - ref).abs() - step - bound).max().item()
    assert worst <= 0, f"off by {worst} more than the bound"


def operands(rows, dim, dtype, kind, post, gates, seed=0, weights=None, bias=0.3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = TYPES[weights or dtype]
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    t = {"x": r(rows, dim).to(TYPES[dtype]), "block": (2 * r(rows, dim) + bias).to(TYPES[dtype]),
         "pre_weight": (1 + 0.2 * r(dim)).to(w)}
    if kind == "layer":
        t["pre_bias"] = r(dim).to(w)
    if post:
        t["post_weight"] = (1 + 0.2 * r(dim)).to(w)
        if kind == "layer":
            t["post_bias"] = r(dim).to(w)
    if gates:
        t["gate"] = r(gates, dim).to(w)
    return t


def run(t, dtype, kind, post, per, scale=0.7, eps=1e-5, want_h=True):
    from emmyrt.norms import ResidualNorm
    op = ResidualNorm(t["x"].shape[1], kind=kind, eps=eps, scale=scale, post_norm=post)
    y, h = torch.empty_like(t["x"]), torch.empty_like(t["x"]) if want_h else None
    op(t["x"], t["block"], y, h, **{n: v for n, v in t.items() if n not in ("x", "block")},
       rows_per_gate=per if "gate" in t else None, stream=torch.cuda.current_stream().cuda_stream)
    return y, h


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 2), (5, 63), (130, 64), (9, 65), (4, 127), (7, 498), (33, 1001), (2, 4096),
                                      (3, 8192), (2, 8193), (3, 8194), (2, 16383), (2, 16384)])
def test_rows(runtime, dtype, kind, rows, dim):
    t = operands(rows, dim, dtype, kind, True, 2)
    per = -(-rows // 2)
    y, h = run(t, dtype, kind, True, per)
    ry, ty, rh, th = reference(t, kind, 1e-5, 0.7, True, per)
    close(y, ry, ty, TYPES[dtype])
    close(h, rh, th, TYPES[dtype])


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gates,per", [(0, 1), (1, 40), (40, 1), (6, 7)])
@pytest.mark.parametrize("weights", ["f32", "bf16", "f16"])
def test_options(runtime, post, gates, per, weights):
    t = operands(40, 1032, "bf16", "layer", post, gates, weights=weights)
    for drop in ((), ("pre_weight", "post_bias"), ("pre_bias", "post_weight")):
        s = {n: v for n, v in t.items() if n not in drop}
        y, h = run(s, "bf16", "layer", post, per)
        ry, ty, rh, th = reference(s, "layer", 1e-5, 0.7, post, per)
        close(y, ry, ty, torch.bfloat16)
        close(h, rh, th, torch.bfloat16)


def test_without_h_and_no_rows(runtime):
    t = operands(6, 100, "f16", "rms", True, 0)
    del t["pre_weight"]
    y, _ = run(t, "f16", "rms", True, 1, want_h=False)
    ry, ty, _, _ = reference(t, "rms", 1e-5, 0.7, True, 1)
    close(y, ry, ty, torch.float16)
    empty = {n: v[:0] for n, v in t.items() if n in ("x", "block")}
    run(empty, "f16", "rms", True, 1)


def test_strides_and_in_place(runtime):
    """Rows of wider buffers, at an odd element too; y over x and h over block; the gaps stay as they are."""
    from emmyrt.norms import ResidualNorm
    for shift in (0, 1, 8):
        wide = torch.randn(4, 12, 320, device="cuda").to(torch.bfloat16)
        before = wide.clone()
        x, block = wide[0, :, shift:shift + 264], wide[1, :, shift:shift + 264]
        w = 1 + 0.1 * torch.randn(264, device="cuda")
        ry, ty, rh, th = reference({"x": x.clone(), "block": block.clone(), "pre_weight": w}, "rms", 1e-6, 2.0, True, 1)
        ResidualNorm(264, scale=2.0)(x, block, x, block, pre_weight=w, stream=torch.cuda.current_stream().cuda_stream)
        close(x, ry, ty, torch.bfloat16)
        close(block, rh, th, torch.bfloat16)
        x.copy_(before[0, :, shift:shift + 264])
        block.copy_(before[1, :, shift:shift + 264])
        assert torch.equal(wide, before)


def test_large_mean_keeps_its_variance(runtime):
    """Values about 3000 that differ by 1: a difference of two sums of squares would lose the variance in f32."""
    x = torch.zeros(4, 777, device="cuda")
    block = 3000 + torch.randn(4, 777, device="cuda")
    t = {"x": x, "block": block}
    y, h = run(t, "f32", "layer", True, 1, scale=1.0)
    ry, ty, rh, th = reference(t, "layer", 1e-5, 1.0, True, 1)
    close(y, ry, ty, torch.float32)
    close(h, rh, th, torch.float32)


def test_zeros_and_not_finite(runtime):
    x = torch.zeros(4, 96, device="cuda")
    block = torch.zeros(4, 96, device="cuda")
    block[1, 5], block[2, 7] = float("inf"), float("nan")
    y, h = run({"x": x, "block": block}, "f32", "rms", True, 1)
    assert (y[[0, 3]] == 0).all() and (h[[0, 3]] == 0).all()      # eps alone under the root
    assert y[1, 5].isnan() and (y[1, :5] == 0).all()              # inf / inf; finite / inf
    assert y[2].isnan().all() and h[1].isnan().all() and h[2].isnan().all()


def test_graph_and_stream(runtime):
    """Captured once and replayed on new values, on a stream of the caller's."""
    from emmyrt.norms import ResidualNorm
    t = operands(37, 520, "bf16", "rms", True, 1)
    op = ResidualNorm(520, scale=0.5)
    y, h = torch.empty_like(t["x"]), torch.empty_like(t["x"])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        for a, b in ((t["x"], y), (y, h)):      # the second call reads the first one's y
            op(a, t["block"], b, post_weight=t["post_weight"], gate=t["gate"], stream=torch.cuda.current_stream().cuda_stream)
    for seed in (1, 2):
        new = operands(37, 520, "bf16", "rms", True, 1, seed)
        for n in t:
            t[n].copy_(new[n])
        g.replay()
        torch.cuda.synchronize()
        ry, ty, _, _ = reference({**new, "pre_weight": None}, "rms", 1e-6, 0.5, True, 37)
        close(y, ry, ty, torch.bfloat16)
        rh, th, _, _ = reference({**new, "x": y, "pre_weight": None}, "rms", 1e-6, 0.5, True, 37)
        close(h, rh, th, torch.bfloat16)


@pytest.mark.parametrize("dim", [64, 65, 1032])
def test_one_row_for_all(runtime, dim):
    """x or block broadcast over the rows (stride 0)."""
    from emmyrt.norms import ResidualNorm
    t = operands(9, dim, "bf16", "rms", True, 0)
    for name in ("x", "block"):
        s = {**t, name: t[name][:1].expand(9, dim)}
        y, h = (torch.empty(9, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        ResidualNorm(dim, eps=1e-5, scale=0.7)(s["x"], s["block"], y, h, post_weight=s["post_weight"], pre_weight=s["pre_weight"],
                                               stream=torch.cuda.current_stream().cuda_stream)
        ry, ty, rh, th = reference(s, "rms", 1e-5, 0.7, True, 9)
        close(y, ry, ty, torch.bfloat16)
        close(h, rh, th, torch.bfloat16)
