"""The operators of a served decoder layer, measured: the block-scaled FP8 linear map, the residual norm,
rotary positions, and appending to and attending over a 4-bit key / value cache.

``run`` computes each one either in plain torch operations (``own`` false) or through ``emmyrt``
(``own`` true), on the same inputs.
"""

import math
import sys
from pathlib import Path

import torch

own = False

TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
BLOCK = 128                 # columns (and weight rows) that share one FP8 scale
E4M3_MAX = 448.0


def listed():
    return [
        # one token through a square projection: bound by the weights' bytes and the launch
        dict(name="linear_1", op="linear", m=1, n=4096, k=4096, dtype="bf16"),
        # a ragged prompt through a down projection whose last blocks of N and K are short
        dict(name="linear_517_odd", op="linear", m=517, n=4112, k=14320, dtype="bf16"),
        # a large prefill batch: bound by the tensor cores
        dict(name="linear_8192", op="linear", m=8192, n=8192, k=8192, dtype="bf16"),
        # a small decode batch: one row per sequence, latency counts
        dict(name="norm_8", op="norm", rows=8, dim=4096, kind="rms", dtype="f16", post=True, gate="channel"),
        # a prefill batch with one gate row per sequence, layer norms with biases
        dict(name="norm_8192", op="norm", rows=8192, dim=4096, kind="layer", dtype="bf16", post=True, gate="sequence"),
        # decode: one token per sequence at far positions, frequencies scaled by parts
        dict(name="rotary_8", op="rotary", tokens=8, q_heads=32, kv_heads=8, dim=128, rotary=128, layout="half",
             scaling="parts", factor=32.0, far=1 << 20, inverse=False, dtype="bf16"),
        # the gradient of a prefill batch, half of each head rotated, interleaved pairs
        dict(name="rotary_16384_grad", op="rotary", tokens=16384, q_heads=32, kv_heads=8, dim=128, rotary=64,
             layout="interleaved", scaling="none", factor=1.0, far=1 << 17, inverse=True, dtype="bf16"),
        # one new token for each of eight sequences
        dict(name="append_8", op="append", tokens=8, kv_heads=8, dim=128, page=64, pages=64, dtype="bf16"),
        # a prompt's keys and values written to their pages
        dict(name="append_16384", op="append", tokens=16384, kv_heads=8, dim=128, page=16, pages=2048, dtype="bf16"),
        # one short sequence, one new token
        dict(name="attend_1x1000", op="attend", batch=1, tokens=1, q_heads=32, kv_heads=8, dim=128, page=64,
             longest=1000, dtype="bf16"),
        # a batch of ragged sequences, some verifying several drafted tokens
        dict(name="attend_16x5000_t3", op="attend", batch=16, tokens=3, q_heads=20, kv_heads=4, dim=64, page=48,
             longest=5000, dtype="f16"),
        # a full decode batch of long sequences
        dict(name="attend_64x16384", op="attend", batch=64, tokens=1, q_heads=32, kv_heads=8, dim=128, page=64,
             longest=16384, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "norm", "rotary", "append", "attend"])
    dtype = rng.choice(["bf16", "f16"])
    if op == "linear":
        m, n, k = _log(rng, 1, 8192), _log(rng, 64, 14336), _log(rng, 64, 14336)
        while m * n * k > 8192 ** 3:
            m = max(1, m // 2)
        return dict(op=op, m=m, n=n, k=k, dtype=dtype)
    if op == "norm":
        dim = _log(rng, 64, 16384)
        rows = min(_log(rng, 1, 65536), max(1, (8192 * 4096) // dim))
        return dict(op=op, rows=rows, dim=dim, kind=rng.choice(["rms", "layer"]),
                    dtype=rng.choice(["bf16", "f16", "f32"]), post=rng.random() < 0.7,
                    gate=rng.choice(["none", "channel", "sequence"]))
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    q_heads = kv_heads * rng.choice([1, 2, 4, 5, 8])
    dim = rng.choice([64, 128])
    if op == "rotary":
        return dict(op=op, tokens=_log(rng, 1, 16384), q_heads=q_heads, kv_heads=kv_heads, dim=dim,
                    rotary=rng.choice([dim, dim // 2, dim // 4]), layout=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "base", "parts"]), factor=rng.choice([4.0, 8.0, 32.0]),
                    far=1 << rng.randrange(12, 21), inverse=rng.random() < 0.5,
                    dtype=rng.choice(["bf16", "f16", "f32"]))
    page = rng.choice([16, 24, 64, 128])
    if op == "append":
        tokens = _log(rng, 1, 16384)
        return dict(op=op, tokens=tokens, kv_heads=kv_heads, dim=dim, page=page, pages=-(-2 * tokens // page) + 1,
                    dtype=dtype)
    batch = _log(rng, 1, 64)
    return dict(op=op, batch=batch, tokens=rng.choice([1, 1, 1, 2, 4, 7]), q_heads=q_heads, kv_heads=kv_heads, dim=dim,
                page=page, longest=_log(rng, 16, 16384), dtype=dtype)


# ---------------------------------------------------------------------------
# inputs


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _emmyrt():
    package = str(Path(__file__).resolve().parents[1] / "emmy-hackathon-2026_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import emmyrt
    emmyrt.init(torch.cuda.current_device())
    return emmyrt


def prepare(case, seed):
    g = _gen(seed)
    return {"linear": _prepare_linear, "norm": _prepare_norm, "rotary": _prepare_rotary, "append": _prepare_append,
            "attend": _prepare_attend}[case["op"]](case, g)


def _prepare_linear(case, g):
    m, n, k = case["m"], case["n"], case["k"]
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    x = _randn(g, m, k)
    x[:, ::97] *= 8.0                                   # a few loud channels, as activations have
    x = x.to(TORCH[case["dtype"]])
    # a quantised checkpoint: e4m3 weights in rows of a multiple of 16 bytes, one scale per 128 x 128 block
    pitch = -(-k // 16) * 16
    wq = torch.zeros(n, pitch, dtype=torch.float8_e4m3fn, device="cuda")
    w = _randn(g, n, k)
    wq[:, :k] = (w * (E4M3_MAX / 6.0)).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    ws = (0.5 + torch.rand(nb, kb, generator=g, device="cuda")) * (6.0 / E4M3_MAX / math.sqrt(k))
    s = dict(op="linear", x=x, wq=wq[:, :k], ws=ws, y=torch.empty(m, n, dtype=x.dtype, device="cuda"))
    if own:
        _emmyrt()
        from emmyrt.blockfp8 import BlockFp8Linear
        s["linear"] = BlockFp8Linear(s["wq"], s["ws"], max_rows=m)
    return s


def _prepare_norm(case, g):
    rows, dim, t = case["rows"], case["dim"], TORCH[case["dtype"]]
    layer = case["kind"] == "layer"
    s = dict(op="norm", kind=case["kind"], eps=1e-6, scale=0.8, post_norm=case["post"],
             x=(3.0 * _randn(g, rows, dim)).to(t), block=(1.5 * _randn(g, rows, dim) + 0.2).to(t))
    s["pre_weight"] = (1.0 + 0.1 * _randn(g, dim)).to(t)
    s["pre_bias"] = (0.1 * _randn(g, dim)).to(t) if layer else None
    s["post_weight"] = (1.0 + 0.1 * _randn(g, dim)).to(t) if case["post"] else None
    s["post_bias"] = (0.1 * _randn(g, dim)).to(t) if case["post"] and layer else None
    s["gate"] = None
    s["rows_per_gate"] = rows
    if case["gate"] == "channel":
        s["gate"] = (0.5 * _randn(g, 1, dim)).to(t)
    elif case["gate"] == "sequence":
        s["rows_per_gate"] = per = max(1, rows // 5)
        s["gate"] = (0.5 * _randn(g, -(-rows // per), dim)).to(t)
    s["y"], s["h"] = torch.empty_like(s["x"]), torch.empty_like(s["x"])
    if own:
        _emmyrt()
        from emmyrt.norms import ResidualNorm
        s["norm"] = ResidualNorm(dim, kind=s["kind"], eps=s["eps"], scale=s["scale"], post_norm=s["post_norm"])
    return s


def _prepare_rotary(case, g):
    t, n, dim = TORCH[case["dtype"]], case["tokens"], case["dim"]
    s = dict(op="rotary", layout=case["layout"], rotary=case["rotary"], scaling=case["scaling"], factor=case["factor"],
             inverse=case["inverse"], base=10000.0, original=4096,
             q=_randn(g, n, case["q_heads"], dim).to(t), k=_randn(g, n, case["kv_heads"], dim).to(t))
    # consecutive positions from a far start, as a chunk of a long sequence has
    start = int(torch.randint(0, case["far"], (1,), generator=g, device="cuda"))
    s["positions"] = (start + torch.arange(n, device="cuda")).to(torch.int32)
    s["q_out"], s["k_out"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
    if own:
        _emmyrt()
        from emmyrt.rotary import Rotary
        s["rope"] = Rotary(dim, rotary_dim=s["rotary"], base=s["base"], layout=s["layout"], scaling=s["scaling"],
                           factor=s["factor"], original_length=s["original"])
    return s


def _cache_arrays(pages, heads, page, dim):
    return dict(k=torch.zeros(pages, heads, page, dim // 2, dtype=torch.uint8, device="cuda"),
                v=torch.zeros(pages, heads, page, dim // 2, dtype=torch.uint8, device="cuda"),
                k_meta=torch.zeros(pages, heads, page, 2, dtype=torch.float16, device="cuda"),
                v_meta=torch.zeros(pages, heads, page, 2, dtype=torch.float16, device="cuda"))


def _cache(a):
    _emmyrt()
    from emmyrt.cache4 import Cache4
    return Cache4(a["k"], a["k_meta"], a["v"], a["v_meta"])


def _prepare_append(case, g):
    n, heads, dim, t = case["tokens"], case["kv_heads"], case["dim"], TORCH[case["dtype"]]
    s = dict(op="append", page=case["page"], arrays=_cache_arrays(case["pages"], heads, case["page"], dim),
             k=_randn(g, n, heads, dim).to(t), v=(0.5 * _randn(g, n, heads, dim)).to(t))
    s["slots"] = torch.randperm(case["pages"] * case["page"], generator=g, device="cuda")[:n].contiguous()
    s["k_stored"], s["v_stored"] = torch.empty_like(s["k"]), torch.empty_like(s["v"])
    if own:
        s["cache"] = _cache(s["arrays"])
    return s


def _prepare_attend(case, g):
    b, page, heads, dim, longest = case["batch"], case["page"], case["kv_heads"], case["dim"], case["longest"]
    t = TORCH[case["dtype"]]
    per = -(-longest // page)
    arrays = _cache_arrays(b * per, heads, page, dim)
    for name in ("k", "v"):
        arrays[name].random_(0, 256, generator=g)
        span = 3.0 + 2.0 * torch.rand(arrays[name].shape[:3], generator=g, device="cuda")
        if name == "v":
            span *= 0.5
        # the levels lie about zero: the least is near minus half the span, 15 steps make the span
        arrays[name + "_meta"][..., 0] = span / 15.0
        arrays[name + "_meta"][..., 1] = -span * (0.4 + 0.2 * torch.rand(span.shape, generator=g, device="cuda"))
    # lengths from a quarter of the longest up; the longest itself is among them
    lengths = (longest * (0.25 + 0.75 * torch.rand(b, generator=g, device="cuda"))).to(torch.int32).clamp(min=1)
    lengths[0] = longest
    s = dict(op="attend", page=page, arrays=arrays, lengths=lengths, scale=dim ** -0.5,
             table=torch.randperm(b * per, generator=g, device="cuda").to(torch.int32).view(b, per),
             q=_randn(g, b, case["tokens"], case["q_heads"], dim).to(t))
    s["out"] = torch.empty_like(s["q"])
    if own:
        cache = _cache(arrays)
        from emmyrt.cache4 import Cache4Attention
        s["attention"] = Cache4Attention(cache, q_heads=case["q_heads"])
    return s


# ---------------------------------------------------------------------------
# one pass


def run(state):
    return {"linear": _linear, "norm": _norm, "rotary": _rotary, "append": _append, "attend": _attend}[state["op"]](state)


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _linear(s):
    if own:
        s["linear"](s["x"], s["y"], stream=_stream())
        return s["y"]
    x, ws = s["x"], s["ws"]
    m, k = x.shape
    n = s["wq"].shape[0]
    kb = ws.shape[1]
    xp = torch.nn.functional.pad(x.float(), (0, kb * BLOCK - k)).view(m, kb, BLOCK)
    amax = xp.abs().amax(-1, keepdim=True)
    scale = amax / torch.full_like(amax, E4M3_MAX)      # a tensor divisor: a true division
    scale = torch.where(scale > 0, scale, torch.ones_like(scale))
    xd = ((xp / scale).to(torch.float8_e4m3fn).float() * scale).view(m, kb * BLOCK)[:, :k]
    wd = s["wq"].float() * ws.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    return (xd @ wd.t()).to(x.dtype)


def _normalised(v, kind, eps, weight, bias):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + eps)
    if weight is not None:
        v = v * weight.float()
    return v if bias is None else v + bias.float()


def _norm(s):
    if own:
        s["norm"](s["x"], s["block"], s["y"], s["h"], post_weight=s["post_weight"], post_bias=s["post_bias"], gate=s["gate"],
                  rows_per_gate=s["rows_per_gate"], pre_weight=s["pre_weight"], pre_bias=s["pre_bias"], stream=_stream())
        return {"y": s["y"], "h": s["h"]}
    x, b = s["x"].float(), s["block"].float()
    if s["post_norm"]:
        b = _normalised(b, s["kind"], s["eps"], s["post_weight"], s["post_bias"])
    if s["gate"] is not None:
        rows = torch.arange(x.shape[0], device=x.device) // s["rows_per_gate"]
        b = b * s["gate"].float()[rows]
    y = x + s["scale"] * b
    h = _normalised(y, s["kind"], s["eps"], s["pre_weight"], s["pre_bias"])
    return {"y": y.to(s["x"].dtype), "h": h.to(s["x"].dtype)}


def _frequencies(s):
    """Radians per position of each pair, in 64 bits, and the factor on the rotated pairs."""
    d, base, factor, magnitude = s["rotary"], s["base"], s["factor"], 1.0
    if s["scaling"] == "base":                          # a larger base: the slowest pair turns `factor` times slower
        base = base * factor ** (d / (d - 2))
    f = base ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
    if s["scaling"] == "linear":
        f = f / factor
    elif s["scaling"] == "parts":
        # pairs that turn over 32 times in the original length keep their frequency, those that turn less than
        # once are slowed by `factor`, those between are mixed
        turns = s["original"] * f / (2 * math.pi)
        keep = ((turns - 1.0) / 31.0).clamp(0, 1)
        f = f / factor * (1 - keep) + f * keep
        magnitude = 0.1 * math.log(factor) + 1.0
    return f, magnitude


def _rotated(s, x, cos, sin):
    r, v = s["rotary"], x.float()
    if s["layout"] == "half":
        a, b = v[..., : r // 2], v[..., r // 2: r]
    else:
        a, b = v[..., 0:r:2], v[..., 1:r:2]
    ra, rb = a * cos - b * sin, a * sin + b * cos
    turned = torch.cat((ra, rb), -1) if s["layout"] == "half" else torch.stack((ra, rb), -1).flatten(-2)
    return torch.cat((turned, v[..., r:]), -1).to(x.dtype)


def _rotary(s):
    if own:
        s["rope"](s["positions"], s["q"], s["k"], q_out=s["q_out"], k_out=s["k_out"], inverse=s["inverse"],
                  stream=_stream())
        return {"q": s["q_out"], "k": s["k_out"]}
    f, magnitude = _frequencies(s)
    angle = s["positions"].double()[:, None, None] * f
    cos, sin = (angle.cos() * magnitude).float(), (angle.sin() * magnitude).float()
    if s["inverse"]:
        sin = -sin
    return {"q": _rotated(s, s["q"], cos, sin), "k": _rotated(s, s["k"], cos, sin)}


def _quantised(x):
    """4-bit levels of each head's vector and its (step, least), both rounded to f16."""
    v = x.float()
    least = v.amin(-1, keepdim=True).to(torch.float16)
    span = v.amax(-1, keepdim=True) - v.amin(-1, keepdim=True)
    step = (span / torch.full_like(span, 15.0)).to(torch.float16)
    s, z = step.float(), least.float()
    level = torch.where(s > 0, (v - z) / torch.where(s > 0, s, torch.ones_like(s)), torch.zeros_like(v))
    return level.round().clamp(0, 15), step, least


def _append(s):
    if own:
        s["cache"].append(s["k"], s["v"], s["slots"], k_stored=s["k_stored"], v_stored=s["v_stored"], stream=_stream())
        return {"k": s["k_stored"], "v": s["v_stored"]}
    page, off = s["slots"] // s["page"], s["slots"] % s["page"]
    out = {}
    for name in ("k", "v"):
        level, step, least = _quantised(s[name])
        n = level.to(torch.uint8)
        s["arrays"][name][page, :, off] = n[..., 0::2] | (n[..., 1::2] << 4)
        s["arrays"][name + "_meta"][page, :, off] = torch.cat((step, least), -1)
        out[name] = (level * step.float() + least.float()).to(s[name].dtype)
    return out


def _dequantised(s, name):
    """[batch, kv heads, positions, dim] in 32 bits, of every position that the page table reaches."""
    packed, meta = s["arrays"][name][s["table"].long()], s["arrays"][name + "_meta"][s["table"].long()].float()
    b, per, heads, page, half = packed.shape
    n = torch.stack((packed & 15, packed >> 4), -1).view(b, per, heads, page, 2 * half).float()
    return (n * meta[..., 0:1] + meta[..., 1:2]).permute(0, 2, 1, 3, 4).reshape(b, heads, per * page, 2 * half)


def _attend(s):
    if own:
        s["attention"](s["q"], s["out"], s["table"], s["lengths"], scale=s["scale"], stream=_stream())
        return s["out"]
    b, t, q_heads, dim = s["q"].shape
    kv = s["arrays"]["k"].shape[1]
    k = _dequantised(s, "k")
    q = s["q"].float().view(b, t, kv, q_heads // kv, dim).permute(0, 2, 1, 3, 4).reshape(b, kv, -1, dim)
    score = (q @ k.transpose(-1, -2)) * s["scale"]
    del k
    # query i of t stands at position length - t + i and sees the keys up to its own; one that stands before the
    # sequence's start sees nothing and gives zeros
    sees = s["lengths"].long()[:, None] - t + 1 + torch.arange(t, device="cuda")
    hidden = torch.arange(score.shape[-1], device="cuda") >= sees.repeat_interleave(q_heads // kv, 1)[:, None, :, None]
    score = score.masked_fill(hidden, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    o = (p @ _dequantised(s, "v")) / torch.where(total > 0, total, torch.ones_like(total))
    return o.view(b, kv, t, q_heads // kv, dim).permute(0, 2, 1, 3, 4).reshape(b, t, q_heads, dim).to(s["q"].dtype)


# ---------------------------------------------------------------------------
# what a pass cannot do without


def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": e * m * (k + n) + n * k + 4 * -(-n // BLOCK) * -(-k // BLOCK), "flops": 2 * m * n * k}
    if case["op"] == "norm":
        return {"bytes": 4 * e * case["rows"] * case["dim"], "flops": 12 * case["rows"] * case["dim"]}
    if case["op"] == "rotary":
        n = case["tokens"] * (case["q_heads"] + case["kv_heads"])
        return {"bytes": 2 * e * n * case["dim"] + 4 * case["tokens"], "flops": 3 * n * case["rotary"]}
    if case["op"] == "append":
        n = 2 * case["tokens"] * case["kv_heads"]
        return {"bytes": n * (2 * e * case["dim"] + case["dim"] // 2 + 4) + 8 * case["tokens"], "flops": 6 * n * case["dim"]}
    # lengths are 5/8 of the longest on average
    length = case["longest"] * (case["batch"] * 0.625 + 0.375)
    return {"bytes": int(length * case["kv_heads"] * 2 * (case["dim"] // 2 + 4)) +
            2 * e * case["batch"] * case["tokens"] * case["q_heads"] * case["dim"],
            "flops": int(4 * length * case["tokens"] * case["q_heads"] * case["dim"])}


# ---------------------------------------------------------------------------
# the definitions in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return {"linear": _exact_linear, "norm": _exact_norm, "rotary": _exact_rotary, "append": _exact_append,
            "attend": _exact_attend}[case["op"]](s)


def _exact_linear(s):
    # the quantisation is part of the operator (f32 scale, nearest e4m3); the sums are in 64 bits, block by block
    x, wq, ws = s["x"].float(), s["wq"], s["ws"].double()
    y = torch.zeros(x.shape[0], wq.shape[0], dtype=torch.float64, device="cuda")
    for b in range(ws.shape[1]):
        xb, wb = x[:, b * BLOCK:(b + 1) * BLOCK], wq[:, b * BLOCK:(b + 1) * BLOCK].double()
        scale = xb.abs().max(1).values.div(torch.tensor(E4M3_MAX, device="cuda").expand(x.shape[0]))
        scale[scale == 0] = 1.0
        q = xb.div(scale[:, None]).to(torch.float8_e4m3fn).double()
        rows = torch.arange(wq.shape[0], device="cuda") // BLOCK
        y += (q @ wb.T) * scale.double()[:, None] * ws[rows, b][None, :]
    return y


def _exact_norm(s):
    def norm(v, weight, bias):
        mean = v.sum(1, keepdim=True) / v.shape[1] if s["kind"] == "layer" else 0.0
        var = ((v - mean) ** 2).sum(1, keepdim=True) / v.shape[1]
        v = (v - mean) / (var + s["eps"]) ** 0.5
        v = v if weight is None else v * weight.double()
        return v if bias is None else v + bias.double()

    b = s["block"].double()
    b = norm(b, s["post_weight"], s["post_bias"]) if s["post_norm"] else b
    if s["gate"] is not None:
        b = b * s["gate"].double().repeat_interleave(s["rows_per_gate"], 0)[: b.shape[0]]
    y = s["x"].double() + s["scale"] * b
    return {"y": y, "h": norm(y, s["pre_weight"], s["pre_bias"])}


def _exact_rotary(s):
    r, half = s["rotary"], s["rotary"] // 2
    base = s["base"] * (s["factor"] ** (r / (r - 2.0)) if s["scaling"] == "base" else 1.0)
    magnitude, freq = 1.0, []
    for i in range(half):
        f = base ** (-2.0 * i / r)
        if s["scaling"] == "linear":
            f /= s["factor"]
        if s["scaling"] == "parts":
            keep = min(1.0, max(0.0, (s["original"] / (2.0 * math.pi / f) - 1.0) / 31.0))
            f = (1.0 - keep) * f / s["factor"] + keep * f
            magnitude = 1.0 + 0.1 * math.log(s["factor"])
        freq.append(f)
    angle = torch.outer(s["positions"].double(), torch.tensor(freq, dtype=torch.float64, device="cuda"))
    turn = torch.polar(torch.full_like(angle, magnitude), -angle if s["inverse"] else angle)[:, None, :]

    def rotate(x):
        v = x.double().clone()
        if s["layout"] == "half":
            z = torch.complex(v[..., :half].contiguous(), v[..., half:r].contiguous()) * turn
            v[..., :half], v[..., half:r] = z.real, z.imag
        else:
            z = torch.view_as_complex(v[..., :r].reshape(*v.shape[:-1], half, 2).contiguous()) * turn
            v[..., :r] = torch.view_as_real(z).reshape(*v.shape[:-1], r)
        return v

    return {"q": rotate(s["q"]), "k": rotate(s["k"])}


def _exact_append(s):
    # steps and least values are stored as f16, so their rounding is part of the operator
    def stored(x):
        v = x.double()
        low, high = v.min(-1).values, v.max(-1).values
        step = ((high - low).float() / torch.full_like(low, 15.0, dtype=torch.float32)).to(torch.float16).double()
        low = low.to(torch.float16).double()
        level = ((v - low[..., None]) / step[..., None]).round().clamp(0, 15)
        level[step == 0] = 0.0
        return level * step[..., None] + low[..., None]

    return {"k": stored(s["k"]), "v": stored(s["v"])}


def _exact_attend(s):
    b, t, q_heads, dim = s["q"].shape
    heads = s["arrays"]["k"].shape[1]
    out = torch.zeros(b, t, q_heads, dim, dtype=torch.float64, device="cuda")

    def rows(name, i, n):
        pages = s["table"][i].long()
        bits = s["arrays"][name][pages].transpose(1, 2).reshape(-1, heads, dim // 2)[:n].int()
        meta = s["arrays"][name + "_meta"][pages].transpose(1, 2).reshape(-1, heads, 2)[:n].double()
        v = torch.empty(n, heads, dim, dtype=torch.float64, device="cuda")
        v[..., 0::2], v[..., 1::2] = bits % 16, bits // 16
        return v * meta[..., :1] + meta[..., 1:]

    for i, n in enumerate(s["lengths"].tolist()):
        k, v = rows("k", i, n), rows("v", i, n)
        for j in range(t):
            m = n - t + j + 1
            if m <= 0:
                continue
            q = s["q"][i, j].double().view(heads, q_heads // heads, dim)
            p = torch.softmax(torch.einsum("hgd,nhd->hgn", q, k[:m]) * s["scale"], -1)
            out[i, j] = torch.einsum("hgn,nhd->hgd", p, v[:m]).reshape(q_heads, dim)
    return out
