"""Attention over the 4-bit cache on the B200 against its definition in f64.

Tolerances, for one output element with probabilities p, steps s, levels n and least values z of the values:
half a step of the type; the rounding of p s to f16, 2^-11 of sum p s n (where the result is f16, sum p and sum p z are taken
of the rounded p: 2^-11 of sum p |v - out|), and of everything else 16 of 2^-24 of
sum p (s n + |z|); and the logits: their f32 sums lose at most 2^-23 at each of the 8 products of 16 and in the
scaling, 16 of 2^-23 of scale (s_k sum |q| n_k + |z_k| sum |q|), which moves every p by that much relative (twice: it is in
the denominator too).
"""

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def stream():
    return torch.cuda.current_stream().cuda_stream


def make(pages, heads, page, dim, seed=0, v_span=1.0):
    from emmyrt.cache4 import Cache4
    g = torch.Generator(device="cuda").manual_seed(seed)
    a = {}
    for name, span in (("k", 4.0), ("v", v_span)):
        a[name] = torch.randint(0, 256, (pages, heads, page, dim // 2), generator=g, device="cuda", dtype=torch.uint8)
        width = span * (0.5 + torch.rand(pages, heads, page, generator=g, device="cuda"))
        a[name + "_meta"] = torch.stack((width / 15, -width * torch.rand(width.shape, generator=g, device="cuda")), -1).half()
    return Cache4(a["k"], a["k_meta"], a["v"], a["v_meta"]), a


def vectors(a, name, table, n, page):
    """levels, step, least [n, heads, ..] of one sequence's first n positions, and which of them exist."""
    pos = torch.arange(n, device="cuda")
    pages = table.long()[pos // page]
    exists = (pages >= 0) & (pages < a[name].shape[0])
    pages = pages.clamp(0, a[name].shape[0] - 1)
    bits, meta = a[name][pages, :, pos % page], a[name + "_meta"][pages, :, pos % page].double()
    return torch.stack((bits & 15, bits >> 4), -1).flatten(-2).double(), meta[..., :1], meta[..., 1:], exists


def reference(a, q, table, lengths, page, scale):
    batch, tokens, q_heads, dim = q.shape
    heads = a["k"].shape[1]
    out, bound = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for b in range(batch):
        length = min(int(lengths[b]), table.shape[1] * page)
        if length <= 0:
            continue
        nk, sk, zk, exists = vectors(a, "k", table[b], length, page)
        nv, sv, zv, _ = vectors(a, "v", table[b], length, page)
        for t in range(tokens):
            sees = exists.clone()
            sees[max(0, length - tokens + t + 1):] = False
            if not sees.any():
                continue
            x = q[b, t].double().view(heads, q_heads // heads, dim)
            k, v = (nk * sk + zk)[sees], (nv * sv + zv)[sees]
            logit = torch.einsum("hgd,nhd->hgn", x, k) * scale
            p = torch.softmax(logit, -1)
            out[b, t] = torch.einsum("hgn,nhd->hgd", p, v).reshape(q_heads, dim)
            size = abs(scale) * (torch.einsum("hgd,nhd->hgn", x.abs(), (nk * sk)[sees]) +
                            x.abs().sum(-1, keepdim=True) * zk.abs()[sees][..., 0].t()[:, None])
            moved = p * (2 * 16 * 2.0 ** -23) * size
            big = (nv * sv)[sees]
            if q.dtype == torch.float16:
                away = (v[:, :, None] - out[b, t].view(1, heads, -1, dim)).abs()
                rounding = torch.einsum("hgn,nhgd->hgd", p, away)
            else:
                rounding = torch.einsum("hgn,nhd->hgd", p, big)
            bound[b, t] = (rounding * 2.0 ** -11 +
                           torch.einsum("hgn,nhd->hgd", moved + p * 16 * 2.0 ** -24, big + zv.abs()[sees]) +
                           moved.sum(-1, keepdim=True) * torch.einsum("hgn,nhd->hgd", p, big + zv.abs()[sees])).reshape(q_heads, dim)
    return out, bound


def close(got, ref, bound):
    step = torch.finfo(got.dtype).eps / 2 * ref.abs() + torch.finfo(got.dtype).tiny
    worst = ((got.double() - ref).abs() - step - bound).max().item()
    assert worst <= 0, f"off by {worst} more than the bound"


def check(dtype, dim, heads, group, tokens, page, lengths, seed=0, scale=None, v_span=1.0, q_size=1.0, spoil=None):
    from emmyrt.cache4 import Cache4Attention
    batch, longest = len(lengths), max(1, *lengths)
    per = -(-longest // page)
    cache, a = make(batch * per + 1, heads, page, dim, seed, v_span)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    table = torch.randperm(batch * per + 1, generator=g, device="cuda")[:batch * per].to(torch.int32).view(batch, per)
    if spoil:
        spoil(table, a)
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    q = (q_size * torch.randn(batch, tokens, heads * group, dim, generator=g, device="cuda")).to(TYPES[dtype])
    out = torch.full_like(q, float("nan"))
    Cache4Attention(cache, heads * group)(q, out, table, lens, scale=scale, stream=stream())
    ref, bound = reference(a, q, table, lens.tolist(), page, dim ** -0.5 if scale is None else scale)
    close(out, ref, bound)
    return cache, a, q, table, lens, out


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,group,tokens", [(1, 1, 1), (2, 4, 1), (1, 8, 1), (2, 5, 2), (1, 16, 1), (3, 3, 7), (1, 7, 5)])
@pytest.mark.parametrize("page", [16, 24])
def test_small(runtime, dtype, dim, heads, group, tokens, page):
    check(dtype, dim, heads, group, tokens, page, [1, 0, 15, 16, 17, 31, 127, 128, 129, 300, 2])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lengths", [[70001], [9000] * 3, [1] * 700, [4000, 1, 1, 1, 20000, 0, 128]])
def test_runs(runtime, dim, lengths):
    """One sequence over all blocks, equal ones, more sequences than blocks, ragged ones."""
    check("bf16", dim, 2, 4, 1, 64, lengths)


@pytest.mark.parametrize("page", [1, 7, 128, 1000])
def test_pages(runtime, page):
    check("f16", 128, 2, 2, 1, page, [1, 999, 1000, 1001, 130])


def test_queries_before_the_start(runtime):
    """More queries than positions: those before the sequence's start see nothing and give zeros."""
    *_, out = check("bf16", 64, 2, 4, 6, 16, [3, 6, 0, 1])
    assert (out[0, :3] == 0).all() and (out[2] == 0).all() and (out[3, :5] == 0).all() and (out[1] != 0).any(-1).all()


def test_extreme_sizes(runtime):
    """One key that outweighs all others; tiny values whose steps are subnormal f16; large and tiny queries."""
    check("bf16", 128, 1, 4, 1, 16, [500, 3], scale=30.0)
    check("f16", 128, 1, 4, 1, 16, [500, 3], v_span=2.0 ** -12)
    check("f16", 128, 1, 4, 1, 16, [500, 3], v_span=40000.0 / 2)
    check("bf16", 128, 1, 4, 1, 16, [500, 3], scale=0.0)
    check("bf16", 128, 1, 4, 1, 16, [500, 3], scale=-0.3)
    check("bf16", 64, 1, 4, 1, 16, [500, 3], q_size=2.0 ** 40, scale=2.0 ** -43)
    check("bf16", 64, 1, 4, 1, 16, [500, 3], q_size=2.0 ** -60, scale=2.0 ** 57)


def test_pages_that_are_none(runtime):
    """Entries below zero and past the cache are not seen, at the start, inside and at the end of a sequence."""
    def spoil(table, a):
        table[0, 3], table[1, 0], table[2, -1], table[3, :] = -1, 1 << 30, a["k"].shape[0], -(1 << 31)
    *_, out = check("bf16", 128, 2, 4, 2, 16, [400, 399, 400, 400], spoil=spoil)
    assert (out[3] == 0).all()


def test_not_finite_where_nothing_is_seen(runtime):
    """NaN and infinity behind a sequence's end, in unseen pages and in hidden positions do not reach the result; one that is
    seen does, in its own head and sequence only."""
    def spoil(table, a):
        used = torch.zeros(a["k"].shape[0], dtype=torch.bool, device="cuda")
        used[table.flatten().long()] = True
        for name in ("k_meta", "v_meta"):
            a[name][~used] = float("nan")
            a[name][table[0, 6].long(), :, 4:] = float("nan")          # from position 100 on, where the sequence ends
            a[name][table[1, 6].long(), :, 4:] = float("inf")
    cache, a, q, table, lens, out = check("f16", 64, 2, 4, 1, 16, [100, 100, 180], spoil=spoil)
    a["v_meta"][table[2, 1].long(), 1, 2, 0] = float("nan")
    again = torch.empty_like(out)
    from emmyrt.cache4 import Cache4Attention
    Cache4Attention(cache, 8)(q, again, table, lens, stream=stream())
    assert torch.equal(again[:2], out[:2]) and torch.equal(again[2, :, :4], out[2, :, :4]) and again[2, :, 4:].isnan().all()


def test_lengths_past_the_table(runtime):
    from emmyrt.cache4 import Cache4Attention
    cache, a = make(8, 1, 16, 64)
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    q = torch.randn(2, 1, 2, 64, device="cuda").half()
    outs = []
    for lens in ([64, 64], [1 << 30, 65]):
        outs.append(torch.empty_like(q))
        Cache4Attention(cache, 2)(q, outs[-1], table, torch.tensor(lens, dtype=torch.int32, device="cuda"), stream=stream())
    assert torch.equal(*outs)
    Cache4Attention(cache, 2)(q, outs[0], table[:, :0], torch.tensor([5, 5], dtype=torch.int32, device="cuda"), stream=stream())
    assert (outs[0] == 0).all()
    Cache4Attention(cache, 2)(q[:0], outs[0][:0], table[:0], torch.zeros(0, dtype=torch.int32, device="cuda"), stream=stream())


def test_repeats_and_strides(runtime):
    """The same bits each time, in place and out of a projection's rows, and beside a table with longer rows."""
    from emmyrt.cache4 import Cache4Attention
    cache, a, q, table, lens, out = check("bf16", 128, 2, 4, 3, 16, [700, 33, 5000])
    op = Cache4Attention(cache, 8)
    wide = torch.zeros(3, 3, 8 * 128 + 200, device="cuda", dtype=torch.bfloat16)
    inside = wide[..., 3:3 + 1024].unflatten(-1, (8, 128))
    long_table = torch.full((3, table.shape[1] + 9), -1, dtype=torch.int32, device="cuda")
    long_table[:, :table.shape[1]] = table
    for _ in range(3):
        inside.copy_(q)
        op(inside, inside, long_table[:, :table.shape[1]], lens, stream=stream())
        assert torch.equal(inside, out)
    assert (wide[..., :3] == 0).all() and (wide[..., 1027:] == 0).all()


def test_slots_past_2_to_31_bytes(runtime):
    """A cache whose levels pass 2^32 bytes: offsets are 64-bit."""
    from emmyrt.cache4 import Cache4, Cache4Attention
    pages, heads, page, dim = 70000, 8, 128, 128
    k, v = (torch.zeros(pages, heads, page, dim // 2, dtype=torch.uint8, device="cuda") for _ in range(2))
    km, vm = (torch.zeros(pages, heads, page, 2, dtype=torch.float16, device="cuda") for _ in range(2))
    cache = Cache4(k, km, v, vm)
    x = torch.randn(2, heads, dim, device="cuda").half()
    y = torch.empty_like(x)
    cache.append(x, x, torch.tensor([pages * page - 1, (pages - 1) * page], device="cuda"), v_stored=y, stream=stream())
    q = torch.randn(1, 1, heads, dim, device="cuda").half()
    out = torch.empty_like(q)
    Cache4Attention(cache, heads)(q, out, torch.tensor([[pages - 1]], dtype=torch.int32, device="cuda"),
                                  torch.ones(1, dtype=torch.int32, device="cuda"), stream=stream())
    # one position: its value, whose p s is rounded to f16 like any other
    assert ((out[0, 0].float() - y[1].float()).abs() <= 2.0 ** -10 * 16 * (y[1].float().abs().amax() / 7) + 2.0 ** -11 * y[1].float().abs()).all()


def test_graph(runtime):
    """Append and attention captured together and replayed while the sequences grow."""
    from emmyrt.cache4 import Cache4Attention
    cache, a = make(64, 2, 16, 64)
    table = torch.randperm(64, device="cuda").to(torch.int32).view(4, 16)
    lens = torch.tensor([5, 100, 0, 250], dtype=torch.int32, device="cuda")
    q, k, v = (torch.zeros(4, 1, h, 64, device="cuda", dtype=torch.bfloat16) for h in (8, 2, 2))
    slots = torch.zeros(4, dtype=torch.int64, device="cuda")
    out = torch.empty_like(q)
    op = Cache4Attention(cache, 8)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cache.append(k[:, 0], v[:, 0], slots, stream=stream())
        op(q, out, table, lens, stream=stream())
    for step in range(4):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, device="cuda"))
        slots.copy_(table.long().gather(1, (lens.long() // 16)[:, None])[:, 0] * 16 + lens.long() % 16)
        lens += 1
        g.replay()
        torch.cuda.synchronize()
        ref, bound = reference(a, q, table, lens.tolist(), 16, 0.125)
        close(out, ref, bound)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim,heads,group,tokens,page,lengths", [
    (64, 2, 4, 2, 16, [100, 64, 2, 3000]), (128, 1, 4, 3, 64, [130, 65, 64, 5000]), (64, 1, 1, 7, 24, [127, 129, 7, 700]),
    (128, 2, 2, 5, 16, [63, 128, 5, 2500])])
@pytest.mark.parametrize("part,value", [(0, float("nan")), (1, float("nan")), (0, float("inf")), (1, float("-inf"))])
def test_not_finite_behind_a_query(runtime, dtype, dim, heads, group, tokens, page, lengths, part, value):
    """A key and a value that are not finite at the last position are seen by the last query alone: the earlier ones of the same
    call, which share its tile, give what they give without it."""
    from emmyrt.cache4 import Cache4Attention
    batch, per = len(lengths), -(-max(lengths) // page)
    cache, a = make(batch * per, heads, page, dim, seed=3)
    table = torch.randperm(batch * per, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda").to(torch.int32).view(batch, per)
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    q = torch.randn(batch, tokens, heads * group, dim, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda").to(TYPES[dtype])
    for b, n in enumerate(lengths):
        for name in ("k_meta", "v_meta"):
            a[name][table[b, (n - 1) // page].long(), :, (n - 1) % page, part] = value
    out = torch.full_like(q, 7.0)
    Cache4Attention(cache, heads * group)(q, out, table, lens, stream=stream())
    ref, bound = reference(a, q[:, :-1], table, [n - 1 for n in lengths], page, dim ** -0.5)
    close(out[:, :-1], ref, bound)
    assert not out[:, -1].isfinite().any()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_long_sums_are_not_biased(runtime, dtype):
    """131072 positions of equal probability whose values nearly cancel: a mean of 4-bit levels about its middle.

    All keys are the same, so every p is 1 and p s exactly an f16 number: nothing is left but the sums.  What they lose must not pile
    up over the tiles a block takes in a row (147 here).  Tensor cores drop bits below 2^-22 of the sum at each of the 4 products of
    a tile of 64 tokens, always towards zero: 4 of 2^-22 of sum p s n, whatever the length.  All other sums round to nearest, which
    averages out: the signed error's mean over 128 heads of 128 is allowed 2^-22 of sum p (s n + |z|) for them (a chain of
    1200 additions is off by 0.6 sqrt(1200) 2^-24 = 21 of 2^-24 for one thread, and 128 heads of some 80 threads each take its mean
    below one of 2^-24).  Sums that go through all 590 products of a run are off by 35 times the bound's first part."""
    from emmyrt.cache4 import Cache4, Cache4Attention
    batch, heads, dim, page, length = 8, 16, 128, 128, 131072
    g = torch.Generator(device="cuda").manual_seed(1)
    per = length // page
    k = torch.zeros(batch * per, heads, page, dim // 2, dtype=torch.uint8, device="cuda")
    km = torch.zeros(batch * per, heads, page, 2, dtype=torch.float16, device="cuda")
    v = torch.randint(0, 256, k.shape, generator=g, device="cuda", dtype=torch.uint8)
    step = ((1 + torch.rand(k.shape[:3], generator=g, device="cuda")) / 16).half()
    vm = torch.stack((step, (-7.5 * step.float()).half()), -1)
    table = torch.arange(batch * per, dtype=torch.int32, device="cuda").view(batch, per)
    lens = torch.full((batch,), length, dtype=torch.int32, device="cuda")
    q = torch.randn(batch, 1, heads, dim, generator=g, device="cuda").to(TYPES[dtype])
    out = torch.empty_like(q)
    Cache4Attention(Cache4(k, km, v, vm), heads)(q, out, table, lens, stream=stream())
    error, first, second = 0.0, 0.0, 0.0
    for b in range(batch):
        for h in range(heads):
            bits = v[b * per:(b + 1) * per, h].reshape(length, dim // 2)
            s, z = vm[b * per:(b + 1) * per, h].reshape(length, 2).double().t()[:, :, None]
            for half, n in ((0, bits & 15), (1, bits >> 4)):
                sn = n.double() * s
                error += (out[b, 0, h, half::2].double() - (sn + z).mean(0)).sum().item()
                first += sn.mean(0).sum().item()
                second += (sn.mean(0) + z.abs().mean(0)).sum().item()
    count = batch * heads * dim
    error, first, second = error / count, first / count, second / count
    assert abs(error) <= 4 * 2.0 ** -22 * first + 2.0 ** -22 * second, (error / first, first, second)


@pytest.mark.parametrize("dtype,dim,heads,group,tokens,page,lengths", [
    ("bf16", 128, 2, 4, 33, 64, [33, 500, 20]), ("f16", 64, 1, 5, 128, 48, [700, 128, 129]), ("bf16", 64, 1, 1, 130, 16, [1000, 131]),
    ("f16", 128, 1, 3, 500, 64, [500, 777]), ("bf16", 128, 1, 2, 500, 24, [2100, 400])])
def test_prompts(runtime, dtype, dim, heads, group, tokens, page, lengths):
    """Many queries a sequence, over what the cache holds before them and over each other."""
    check(dtype, dim, heads, group, tokens, page, lengths)
