"""A decoder layer's serving steps made of the operators together: page plan, norm, projections, cache write, attention;
eager, on other streams, captured and replayed, and with caches whose offsets pass 32 bits."""
import pytest

torch = pytest.importorskip("torch")

import serving_plain as plain  # noqa: E402
from test_gpu_parity import pk  # noqa: E402, F401
from test_gpu_paged_attention import Case  # noqa: E402
from test_gpu_serving import check_norm, gen, randn, weights  # noqa: E402

pytestmark = pytest.mark.gpu


class Layer:
    """One layer's attention half for up to `capacity` new tokens of a few requests, in tensors that stay where they are."""

    heads, kv, d, width, page, columns, capacity, eps = 8, 2, 64, 512, 16, 40, 12, 1e-5

    def __init__(self, pk, requests, fp8, seed=3):  # noqa: F811
        g = gen(seed)
        self.pk, self.fp8, self.requests = pk, fp8, requests
        i32 = lambda *shape, fill=0: torch.full(shape, fill, dtype=torch.int32, device="cuda")  # noqa: E731
        pages = requests * self.columns
        self.norm = randn(g, self.width)
        self.qkv_w, self.out_w = weights(g, (self.heads + 2 * self.kv) * self.d, self.width), weights(g, self.width, self.heads * self.d)
        self.bias = torch.randn((self.heads + 2 * self.kv) * self.d, generator=g, device="cuda")
        kind = torch.uint8 if fp8 else torch.float16
        # nothing but what is written may matter: the cache begins as NaN
        self.key = torch.full((pages, self.kv, self.page, self.d), 0x7F if fp8 else float("nan"), dtype=kind, device="cuda")
        self.value = torch.full((pages, self.kv, self.d, self.page), 0x7F if fp8 else float("nan"), dtype=kind, device="cuda")
        self.key_scale, self.value_scale = (0.25, 0.125) if fp8 else (1.0, 1.0)
        self.free = torch.randperm(pages, generator=g, device="cuda").int()
        self.range, self.table = i32(2), i32(requests, self.columns, fill=-1)
        self.range[1] = pages
        self.held, self.added, self.lengths, self.starts = i32(requests), i32(requests), i32(requests), i32(requests + 1)
        self.slots, self.positions, self.info = i32(self.capacity), i32(self.capacity), i32(4)
        half = lambda n: torch.zeros((self.capacity, n), dtype=torch.float16, device="cuda")  # noqa: E731
        self.x, self.residual, self.qkv, self.y = half(self.width), half(self.width), half((self.heads + 2 * self.kv) * self.d), half(self.width)
        self.codes, self.scales = torch.zeros((self.capacity, self.width), dtype=torch.int8, device="cuda"), torch.ones(self.capacity, device="cuda")
        self.o = torch.zeros((self.capacity, self.heads, self.d), dtype=torch.float16, device="cuda")
        size = pk.paged_attention_workspace_bytes(self.capacity, self.capacity, requests, self.heads, self.kv, self.d, self.page, self.columns)
        self.workspace = torch.empty(size, dtype=torch.uint8, device="cuda")

    def parts(self):
        rows = self.qkv.view(self.capacity, -1, self.d)
        return rows[:, :self.heads], rows[:, self.heads:self.heads + self.kv], rows[:, self.heads + self.kv:]

    def step(self, stream=None):
        pk_, (q, k, v) = self.pk, self.parts()
        pk_.page_plan(self.held, self.added, self.free, self.range, self.table, self.starts, self.lengths, self.slots, self.positions, self.info,
                      self.page, stream=stream)
        pk_.rms_norm_quantize(pk_.NORM_INT8, self.x, self.residual, self.norm, self.residual, self.codes, self.scales, self.eps, stream=stream)
        pk_.gemv_int4g128_a8(self.codes, self.scales, *self.qkv_w, self.bias, self.qkv, stream=stream)
        pk_.paged_cache_write(k, v, self.slots, self.key, self.value, 1 / self.key_scale, 1 / self.value_scale, stream=stream)
        pk_.paged_attention(q, self.key, self.value, self.table, self.starts, self.lengths, self.o, self.workspace, max_queries=self.capacity,
                            key_scale=self.key_scale, value_scale=self.value_scale, stream=stream)
        pk_.gemv_int4g128(self.o.view(self.capacity, -1), *self.out_w, None, self.y, stream=stream)

    def ask(self, added, g):
        """The next step's input: what was added before is held now, and its pages are taken from the free ones."""
        self.range[0] += self.info[1]
        self.held.copy_(self.lengths)
        self.added.copy_(torch.tensor(added, dtype=torch.int32))
        self.x.copy_(randn(g, self.capacity, self.width))

    def outputs(self):
        return (self.table, self.starts, self.lengths, self.slots, self.positions, self.info, self.residual, self.codes, self.scales, self.qkv, self.key,
                self.value, self.o, self.y)


STEPS = [[5, 0, 7, 0], [1, 1, 1, 0], [0, 9, 1, 2], [1, 1, 1, 1], [12, 0, 0, 0], [0, 0, 0, 0], [1, 1, 0, 1]]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("columns", [30, 250])
@pytest.mark.parametrize("heads", [2, 4, 8])
def test_layer_steps(pk, fp8, columns, heads):  # noqa: F811
    """Each operator's output against the definition applied to what the one before it left (tables of 480 and of 4000 keys; 12, 24
    and 48 rows a kv head)."""
    layer = type("Sized", (Layer,), {"columns": columns, "heads": heads})(pk, 4, fp8)
    g, held = gen(8), [0] * 4
    for added in STEPS:
        layer.ask(added, g)
        before = [t.clone() for t in (layer.residual, layer.key, layer.value, layer.o, layer.table)]
        begin = int(layer.range[0])
        layer.o.fill_(9)
        layer.step()
        tokens = sum(added)
        lists = plain.plan(held, added, layer.free.tolist(), begin, layer.key.shape[0], before[4].tolist(), layer.page, layer.capacity)
        for got, want in zip((layer.table, layer.starts, layer.lengths, layer.slots, layer.positions, layer.info), lists):
            assert got.tolist() == want
        held = [h + a for h, a in zip(held, added)]
        h, y = plain.rms_norm(layer.x, before[0], layer.norm, layer.eps)
        plain.close(layer.residual, h, h.abs() * (plain.U16 + 2 * plain.U32) + plain.TINY16, "residual")
        rel = (74 / 2 + 6) * plain.U32
        s = layer.scales.double()[:, None]
        plain.close(layer.codes.double() * s, y, 0.5 * s + 2 * rel * y.abs() + s * 1e-6, "codes")
        want, bound = plain.gemv(layer.codes, layer.scales, *layer.qkv_w, layer.bias)
        plain.close(layer.qkv, want, bound + want.abs() * plain.U16 * (1 + 2.0**-10) + plain.TINY16, "projections")
        q, k, v = layer.parts()
        at = layer.slots[:tokens].long()
        enc = lambda x, s: (x[:tokens].float() * (1 / s)).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8) if fp8 else x[:tokens]  # noqa: E731
        before[1][at // layer.page, :, at % layer.page] = enc(k, layer.key_scale)
        before[2].transpose(2, 3)[at // layer.page, :, at % layer.page] = enc(v, layer.value_scale)
        bits = lambda x: x if fp8 else x.view(torch.int16)  # noqa: E731
        assert torch.equal(bits(layer.key), bits(before[1])) and torch.equal(bits(layer.value), bits(before[2]))
        want, bound = plain.attention(q[:tokens], layer.key, layer.value, layer.table, layer.starts, layer.lengths, -1, 0, layer.d**-0.5, layer.key_scale,
                                      layer.value_scale)
        plain.close(layer.o[:tokens], want, bound, "attention")
        assert (layer.o[tokens:] == 9).all()
        want, bound = plain.gemv(layer.o.view(layer.capacity, -1), None, *layer.out_w, None)
        plain.close(layer.y, want, bound + want.abs() * plain.U16 * (1 + 2.0**-10) + plain.TINY16, "output")


@pytest.mark.parametrize("fp8", [False, True])
def test_layer_steps_in_a_graph(pk, fp8):  # noqa: F811
    """Replays equal eager steps bit for bit, with the program's own work between them; two graphs share a workspace in turn."""
    eager, graphed, other = (Layer(pk, 4, fp8) for _ in range(3))
    other.workspace = graphed.workspace
    graphs = []
    for layer in (graphed, other):
        layer.step()  # nothing is asked for yet: no token, no page
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            layer.step()
        graphs.append(graph)
    for layer in (graphed, other):
        for t, u in zip(layer.outputs(), eager.outputs()):
            t.copy_(u)  # as at the start: the steps so far added nothing, but moved the residual
    g, g2, g3 = gen(8), gen(8), gen(8)
    for added in STEPS:
        eager.ask(added, g)
        eager.step()
        graphed.ask(added, g2)
        other.ask(added, g3)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for layer in (graphed, other):
            for got, want in zip(layer.outputs(), eager.outputs()):
                same = lambda t: t.view(torch.int16) if t.dtype is torch.float16 else t  # noqa: E731
                assert torch.equal(same(got), same(want))


@pytest.mark.parametrize("explicit", [False, True])
def test_layer_steps_on_two_streams(pk, explicit):  # noqa: F811
    """Two layers at once on streams of their own, behind work that the streams have yet to do, equal one after the other."""
    streams = [torch.cuda.Stream() for _ in range(2)]
    together, alone = [Layer(pk, 4, False, seed) for seed in (5, 6)], [Layer(pk, 4, False, seed) for seed in (5, 6)]
    torch.cuda.synchronize()
    for layer, g in zip(alone, (gen(1), gen(2))):
        for added in STEPS:
            layer.ask(added, g)
            layer.step()
    torch.cuda.synchronize()
    gens = (gen(1), gen(2))
    for added in STEPS:
        for layer, g, stream in zip(together, gens, streams):
            with torch.cuda.stream(stream):
                torch.cuda._sleep(200000)
                layer.ask(added, g)
                if not explicit:
                    layer.step()
            if explicit:  # from the default stream, named
                layer.step(stream)
    torch.cuda.synchronize()
    for a, b in zip(together, alone):
        for got, want in zip(a.outputs(), b.outputs()):
            same = lambda t: t.view(torch.int16) if t.dtype is torch.float16 else t  # noqa: E731
            assert torch.equal(same(got), same(want))


@pytest.mark.parametrize("n", [1, 3, 40])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("length", [300, 900])
def test_cache_offsets_beyond_32_bits(pk, n, fp8, length):  # noqa: F811
    """Pages at the end of caches of more than 2^32 values (fp16: 2^33 bytes each), written and read there."""
    kv, d, page = 8, 128, 256
    pages = (1 << 32) // (kv * d * page) + 40
    kind = torch.uint8 if fp8 else torch.float16
    key = torch.empty((pages, kv, page, d), dtype=kind, device="cuda")
    value = torch.empty((pages, kv, d, page), dtype=kind, device="cuda")
    g = gen(n + length)
    ids = pages - 1 - torch.randperm(30, generator=g, device="cuda").int()
    columns = -(-length // page)
    table = torch.stack([ids[:columns], ids[columns:2 * columns]])
    at = torch.arange(length, device="cuda")
    slots = torch.cat([table[r][at // page] * page + at % page for r in range(2)]).int()
    rows = randn(g, 2 * length, 2 * kv, d)
    pk.paged_cache_write(rows[:, :kv], rows[:, kv:], slots, key, value)
    stored = rows.float().to(torch.float8_e4m3fn).view(torch.uint8) if fp8 else rows  # |x| < 448
    for r in range(2):
        part, at_r = stored[r * length:(r + 1) * length], slots[r * length:(r + 1) * length].long()
        assert torch.equal(key[at_r // page, :, at_r % page], part[:, :kv])
        assert torch.equal(value[table[r].long()].permute(0, 3, 1, 2).reshape(-1, kv, d)[:length], part[:, kv:])
    q = randn(g, 2 * n, 2 * kv, d)
    starts = torch.tensor([0, n, 2 * n], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([length, length - 7], dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)
    size = pk.paged_attention_workspace_bytes(2 * n, n, 2, 2 * kv, kv, d, page, columns)
    pk.paged_attention(q, key, value, table, starts, lengths, out, torch.empty(size, dtype=torch.uint8, device="cuda") if size else None, max_queries=n)
    want, bound = plain.attention(q, key, value, table, starts, lengths, -1, 0, d**-0.5)
    plain.close(out, want, bound)


@pytest.mark.parametrize("n", [1, 40])
def test_attention_calls_with_their_own_workspaces_at_once(pk, n):  # noqa: F811
    shapes = ([(n, 3000), (1, 40), (n, 900)], [(n, 50), (n, 2500)])
    cases = [Case(shape, heads=8, kv=2, seed=i) for i, shape in enumerate(shapes)]
    want = [case.run(pk).clone() for case in cases]
    torch.cuda.synchronize()
    streams, spaces, outs = [torch.cuda.Stream() for _ in cases], [case.workspace(pk) for case in cases], [torch.full_like(case.out, 9.0) for case in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        for case, stream, space, out in zip(cases, streams, spaces, outs):
            with torch.cuda.stream(stream):
                case.run(pk, workspace=space, out=out)
    torch.cuda.synchronize()
    for out, first in zip(outs, want):
        assert torch.equal(out, first)


def test_norm_of_the_hidden_width(pk):  # noqa: F811
    """The width and rows that the steps above use, by themselves."""
    g = gen(4)
    check_norm(pk, pk.NORM_INT8, randn(g, 12, 512), randn(g, 12, 512), randn(g, 512), 1e-5)
