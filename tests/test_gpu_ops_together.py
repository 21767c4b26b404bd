"""A decoder layer's attention half made of the operators, as a server would call them.

x and the last block's result -> residual norm -> FP8 projection -> rotary on q and k inside the projection's rows -> append to
the 4-bit cache -> attention over it -> FP8 projection -> residual norm.  Each operator is checked against f64 on what it was
given, with its own tolerance (they are in the operators' own tests); the run as a whole has to give the same bits eagerly, from
a captured graph, and beside other calls on another stream.
"""

import threading

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import test_gpu_ops_attend as attend_test      # noqa: E402
import test_gpu_ops_blockfp8 as fp8_test       # noqa: E402
import test_gpu_ops_cache4 as cache_test       # noqa: E402
import test_gpu_ops_norm as norm_test          # noqa: E402
import test_gpu_ops_rotary as rotary_test      # noqa: E402

H, QH, KH, D, PAGE, PAGES, BATCH = 320, 6, 2, 64, 16, 40, 5
EPS = 1e-5


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(seed, *shape):
    return torch.randn(*shape, generator=gen(seed), device="cuda").to(torch.bfloat16)


class Layer:
    """The layer and the buffers of calls of `tokens` tokens for each of BATCH sequences."""

    def __init__(self, tokens, seed=0):
        from emmyrt.blockfp8 import BlockFp8Linear
        from emmyrt.cache4 import Cache4, Cache4Attention
        from emmyrt.norms import ResidualNorm
        from emmyrt.rotary import Rotary
        self.tokens, rows = tokens, BATCH * tokens
        self.weights = {"qkv": fp8_test.weights((QH + 2 * KH) * D, H, seed), "out": fp8_test.weights(H, QH * D, seed + 1)}
        self.norm_weights = (1 + 0.2 * randn(seed + 2, H).float()).to(torch.bfloat16)
        self.parts = {"k": torch.zeros(PAGES, KH, PAGE, D // 2, dtype=torch.uint8, device="cuda"),
                      "k_meta": torch.zeros(PAGES, KH, PAGE, 2, dtype=torch.float16, device="cuda")}
        self.parts.update(v=self.parts["k"].clone(), v_meta=self.parts["k_meta"].clone())
        self.norm, self.rotary = ResidualNorm(H, eps=EPS), Rotary(D, base=50000.0)
        self.qkv_map, self.out_map = (BlockFp8Linear(*self.weights[n], max_rows=rows) for n in ("qkv", "out"))
        self.cache = Cache4(self.parts["k"], self.parts["k_meta"], self.parts["v"], self.parts["v_meta"])
        self.attention = Cache4Attention(self.cache, QH)
        empty = lambda *s: torch.empty(*s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
        self.x, self.block, self.y, self.h = (empty(rows, H) for _ in range(4))
        self.qkv, self.mixed = empty(rows, (QH + 2 * KH) * D), empty(rows, QH * D)
        self.o, self.y2, self.h2 = (empty(rows, H) for _ in range(3))
        self.positions = torch.zeros(rows, dtype=torch.int32, device="cuda")
        self.slots = torch.zeros(rows, dtype=torch.int64, device="cuda")
        self.lengths = torch.zeros(BATCH, dtype=torch.int32, device="cuda")
        # each sequence has 8 pages of its own, in no order
        self.table = torch.randperm(PAGES, generator=gen(seed + 3), device="cuda").view(BATCH, 8).to(torch.int32)
        heads = self.qkv.view(rows, QH + 2 * KH, D)
        self.q, self.k, self.v = heads[:, :QH], heads[:, QH:QH + KH], heads[:, QH + KH:]

    def load(self, before, seed):
        """Inputs of one call; `before` tokens are held of each sequence, and None where the batch has only padding."""
        self.x.copy_(randn(seed, *self.x.shape))
        self.block.copy_(randn(seed + 1, *self.block.shape))
        for b, n in enumerate(before):
            for t in range(self.tokens):
                i, at = b * self.tokens + t, 0 if n is None else n + t
                self.positions[i] = at
                self.slots[i] = -1 if n is None else self.table[b, at // PAGE].long() * PAGE + at % PAGE
            self.lengths[b] = 0 if n is None else n + self.tokens

    def attend_shapes(self):
        return self.q.unflatten(0, (BATCH, self.tokens)), self.mixed.view(BATCH, self.tokens, QH, D)

    def run(self, stream, look=lambda name: None):
        w = self.norm_weights
        q, mixed = self.attend_shapes()
        self.norm(self.x, self.block, self.y, self.h, pre_weight=w, stream=stream)
        self.qkv_map(self.h, self.qkv, stream=stream)
        look("projected")
        self.rotary(self.positions, self.q, self.k, stream=stream)
        self.cache.append(self.k, self.v, self.slots, stream=stream)
        self.attention(q, mixed, self.table, self.lengths, stream=stream)
        self.out_map(self.mixed, self.o, stream=stream)
        self.norm(self.y, self.o, self.y2, self.h2, pre_weight=w, stream=stream)

    def results(self):
        return [t.clone() for t in (self.y, self.h, self.qkv, self.mixed, self.o, self.y2, self.h2, *self.parts.values())]


def check_norm(x, block, y, h, w):
    t = {"x": x, "block": block, "pre_weight": w}
    ry, ty, rh, th = norm_test.reference(t, "rms", EPS, 1.0, True, 1)
    norm_test.close(y, ry, ty, torch.bfloat16)
    norm_test.close(h, rh, th, torch.bfloat16)


def check_product(x, weights, y):
    ref, bound = fp8_test.reference(x, *weights, torch.bfloat16)
    worst = ((y.double() - ref).abs() - bound).max().item()
    assert worst <= 0, f"off by {worst} more than the bound"


def stream_of(s=None):
    return (s or torch.cuda.current_stream()).cuda_stream


@pytest.mark.parametrize("tokens", [1, 2, 19])
def test_every_operator_on_what_it_is_given(runtime, tokens):
    layer = Layer(tokens)
    held = [0, 3, 15, None, 60]
    for name in ("k", "v"):                                # what the cache holds before the call
        layer.parts[name].random_(0, 256, generator=gen(7))
        layer.parts[name + "_meta"].copy_(torch.rand(layer.parts[name + "_meta"].shape, generator=gen(8), device="cuda") * 0.2)
    layer.load(held, 100)
    seen = {}
    before = {n: t.clone() for n, t in layer.parts.items()}
    layer.run(stream_of(), lambda name: seen.update({name: layer.qkv.clone()}))
    check_norm(layer.x, layer.block, layer.y, layer.h, layer.norm_weights)
    check_product(layer.h, layer.weights["qkv"], seen["projected"])
    was = seen["projected"].view(-1, QH + 2 * KH, D)
    rotary_test.close(layer.qkv.view(-1, QH + 2 * KH, D)[:, :QH + KH], was[:, :QH + KH], layer.positions, D, "half", False, base=50000.0)
    assert torch.equal(layer.v, was[:, QH + KH:])
    live = layer.slots >= 0
    slots = layer.slots[live]
    for name, x in (("k", layer.k), ("v", layer.v)):
        n, step, least = cache_test.read(layer.parts, name, slots, PAGE)
        rn, rs, rl = cache_test.quantised(x[live])
        assert torch.equal(step, rs) and torch.equal(least, rl) and torch.equal(n, rn)
    other = torch.ones(PAGES * PAGE, dtype=torch.bool, device="cuda")
    other[slots] = False
    rest = other.nonzero().flatten()
    for name, t in layer.parts.items():
        assert torch.equal(t[rest // PAGE, :, rest % PAGE], before[name][rest // PAGE, :, rest % PAGE])
    q, mixed = layer.attend_shapes()
    ref, bound = attend_test.reference(layer.parts, q, layer.table, layer.lengths, PAGE, D ** -0.5)
    attend_test.close(mixed, ref, bound)
    assert (mixed[3] == 0).all()                           # a row of padding attends to nothing
    check_product(layer.mixed, layer.weights["out"], layer.o)
    check_norm(layer.y, layer.o, layer.y2, layer.h2, layer.norm_weights)
    assert layer.qkv_map.status() == 0 and layer.out_map.status() == 0


def steps(layer, run, count=6):
    """Decodes `count` tokens after a held prefix of zeros; what every step gave."""
    out = []
    held = [0, 13, 31, None, 90]
    for i in range(count):
        layer.load([None if n is None else n + i for n in held], 200 + 2 * i)
        run()
        torch.cuda.synchronize()
        out.append(layer.results())
    return out


def same(a, b):
    assert len(a) == len(b)
    for i, (p, q) in enumerate(zip(a, b)):
        for j, (s, t) in enumerate(zip(p, q)):
            assert torch.equal(s, t), (i, j)


def test_a_graph_captured_with_the_first_call(runtime):
    eager, captured = Layer(1), Layer(1)
    expected = steps(eager, lambda: eager.run(stream_of()))
    captured.load([None] * BATCH, 0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured.run(stream_of())
    same(steps(captured, graph.replay), expected)


def test_two_streams_and_threads(runtime):
    """Two layers with operators of their own, decoding at the same time."""
    layers = [Layer(1, 0), Layer(1, 50)]
    expected = []
    for seed in (0, 50):
        alone = Layer(1, seed)
        expected.append(steps(alone, lambda: alone.run(stream_of())))
    streams = [torch.cuda.Stream() for _ in layers]
    got, errors = [None, None], []

    def work(i):
        try:
            def run():
                with torch.cuda.stream(streams[i]):
                    for _ in range(20):                    # the same call again gives the same
                        layers[i].run(stream_of(streams[i]))
            got[i] = steps(layers[i], lambda: (torch.cuda.current_stream().synchronize(), run()))
        except BaseException as e:      # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for i in range(2):
        same(got[i], expected[i])
