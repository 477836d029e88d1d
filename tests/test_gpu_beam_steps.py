"""Steps of a beam search over a paged cache made of the operators together: page plan, norm and rotation with the write into
the cache, attention, selection, fork of the pages, free list, copies, and histories in their beams' order."""
import pytest

torch = pytest.importorskip("torch")

import decoding_plain as plain  # noqa: E402
import serving_plain  # noqa: E402
from test_gpu_parity import pk  # noqa: E402, F401
from test_gpu_serving import gen, randn  # noqa: E402

pytestmark = pytest.mark.gpu


class Search:
    """One attention layer between an embedding and scores over a small vocabulary, `n` requests of `beams` beams."""

    n, beams, heads, kv, d, page, columns, vocab, width, layers = 3, 4, 4, 2, 64, 16, 6, 200, 64, 2

    def __init__(self, pk, fp8, prompt, seed=3):  # noqa: F811
        g = gen(seed)
        self.pk, self.fp8 = pk, fp8
        rows = self.rows = self.n * self.beams
        i32 = lambda *shape, fill=0: torch.full(shape, fill, dtype=torch.int32, device="cuda")  # noqa: E731
        pages = rows * self.columns
        kind, nan = (torch.uint8, 0x7F) if fp8 else (torch.float16, float("nan"))
        self.key = torch.full((self.layers, pages, self.kv, self.page, self.d), nan, dtype=kind, device="cuda")
        self.value = torch.full((self.layers, pages, self.kv, self.d, self.page), nan, dtype=kind, device="cuda")
        self.inverse = (4.0, 8.0) if fp8 else (1.0, 1.0)
        # queries, keys and values of every token, projected once: a library product of another number of rows may round otherwise
        self.of_token = (randn(g, self.vocab, self.width).float() @ randn(g, self.width, (self.heads + 2 * self.kv) * self.d).float()).half()
        self.of_token, self.out_w = self.of_token.view(self.vocab, -1, self.d), randn(g, self.heads * self.d, self.vocab, scale=0.2)
        self.qw, self.kw, self.words = randn(g, self.d), randn(g, self.d), pk.rotary_frequencies(32)
        self.tables, self.lengths = [i32(rows, self.columns, fill=-1) for _ in range(2)], [i32(rows) for _ in range(2)]
        self.free, self.range = torch.randperm(pages, generator=g, device="cuda").int(), i32(2)
        self.range[1] = pages
        self.capacity = rows * prompt
        self.added, self.starts, self.planned = i32(rows), i32(rows + 1), i32(rows)
        self.slots, self.positions, self.plan_info, self.info = i32(self.capacity), i32(self.capacity), i32(4), i32(4)
        self.copies, self.freed = i32(rows, 2), i32(pages)
        self.q_out = torch.zeros((self.capacity, self.heads, self.d), dtype=torch.float16, device="cuda")
        self.o, self.x = torch.zeros_like(self.q_out), torch.zeros((self.capacity, self.heads + 2 * self.kv, self.d), dtype=torch.float16, device="cuda")
        self.logits = torch.zeros((self.n, self.beams, self.vocab), device="cuda")
        self.scores = torch.full((self.n, self.beams), -float("inf"), device="cuda")
        self.scores[:, 0] = 0  # one beam a request holds the prompt
        self.ended, self.new_ended = (torch.zeros((self.n, self.beams), dtype=torch.bool, device="cuda") for _ in range(2))
        self.new_scores, self.tokens, self.parents = torch.zeros_like(self.scores), i32(self.n, self.beams), i32(self.n, self.beams)
        self.history = i32(self.n, self.beams, 40, fill=-1)
        size = lambda n: torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")  # noqa: E731
        self.attend_space = size(pk.paged_attention_workspace_bytes(self.capacity, prompt, rows, self.heads, self.kv, self.d, self.page, self.columns))
        self.select_space = size(pk.beam_select_workspace_bytes(self.n, self.beams, self.vocab, self.beams))
        self.fork_space = size(pk.page_fork_workspace_bytes(rows, self.columns, pages))
        self.prompt = prompt

    def attend(self, at):
        """New tokens into the cache of both layers (the second holds the same), and their attention."""
        pk_, (q, k, v) = self.pk, (self.x[:, :self.heads], self.x[:, self.heads:self.heads + self.kv], self.x[:, self.heads + self.kv:])
        pk_.page_plan(self.lengths[at], self.added, self.free, self.range, self.tables[at], self.starts, self.planned, self.slots, self.positions,
                      self.plan_info, self.page)
        pk_.page_keep(self.plan_info, None, self.free, self.range)
        for layer in range(self.layers):
            pk_.head_norm_rotary_write(q, k, v, self.qw, self.kw, self.positions, self.slots, self.words, self.q_out, self.key[layer], self.value[layer],
                                       *self.inverse, interleaved=True)
        pk_.paged_attention(self.q_out, self.key[1], self.value[1], self.tables[at], self.starts, self.planned, self.o, self.attend_space,
                            max_queries=self.prompt, key_scale=1 / self.inverse[0], value_scale=1 / self.inverse[1])

    def choose(self, at):
        pk_ = self.pk
        pk_.beam_select(self.logits, self.scores, self.ended, self.new_scores, self.tokens, self.parents, self.new_ended, self.select_space, end_token=7)
        pk_.page_fork(self.parents.view(-1), self.tables[at], self.planned, self.free, self.range, self.tables[1 - at], self.lengths[1 - at], self.copies,
                      self.freed, self.info, self.fork_space, self.page)
        pk_.page_keep(self.info, self.freed, self.free, self.range)
        pk_.paged_cache_copy(self.copies, self.key, self.value)
        pk_.beam_reorder(self.history, self.parents, self.history)

    def outputs(self):
        return (*self.tables, *self.lengths, self.free, self.range, self.slots, self.positions, self.info, self.copies, self.q_out, self.o, self.new_scores,
                self.tokens, self.parents, self.new_ended, self.history, self.key, self.value)

    def begin(self, g):
        """Prompts of different lengths on each request's first row."""
        self.added.zero_()
        lengths = [self.prompt, self.prompt - 5, 1][:self.n]
        self.added[::self.beams] = torch.tensor(lengths, dtype=torch.int32)
        ids = torch.randint(0, self.vocab, (sum(lengths),), generator=g, device="cuda")
        at = 0
        for i, n in enumerate(lengths):
            self.history[i, 0, :n] = ids[at:at + n]
            at += n
        self.feed(ids)

    def feed(self, ids):
        self.x[:len(ids)] = self.of_token[ids]

    def score(self):
        """Scores of each row's last new token."""
        last = (self.starts[1:] - 1).clamp(min=0).long()
        self.logits.copy_((self.o[last].view(self.rows, -1).float() @ self.out_w.float()).view(self.logits.shape))

    def move(self):
        """The chosen tokens are what the next step adds; ended beams add nothing."""
        self.scores.copy_(self.new_scores)
        adds = (self.parents.view(-1) >= 0) & ~self.new_ended.view(-1)
        was = self.ended.view(-1)[self.parents.view(-1).clamp(min=0).long()]
        self.ended.copy_(self.new_ended)
        self.added.copy_(adds.int())
        return adds, was


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("prompt", [16, 21])
def test_beam_search(pk, fp8, prompt):  # noqa: F811
    s, g = Search(pk, fp8, prompt), gen(5)
    s.begin(g)
    histories = [h[h >= 0].tolist() for h in s.history.view(s.rows, -1)]
    forks = 0
    for step in range(18):
        at = step % 2
        s.attend(at)
        # every row's cache is what its own history gives, whatever beams it came from
        lengths = s.planned.tolist()
        assert int(s.plan_info[2]) == 0 and lengths == [len(h) for h in histories]
        for r, h in enumerate(histories):
            if not h:
                continue
            x = s.of_token[torch.tensor(h, device="cuda")]
            k, v = x[:, s.heads:s.heads + s.kv], x[:, s.heads + s.kv:]
            y, bound = plain.head_norm_rotary(k, s.kw, torch.arange(len(h)), s.words, True, 1.0, 1e-6)
            ids, t = s.tables[at][r].long(), torch.arange(len(h), device="cuda")
            for layer in range(s.layers):
                got_k, got_v = s.key[layer][ids[t // s.page], :, t % s.page], s.value[layer].transpose(2, 3)[ids[t // s.page], :, t % s.page]
                if fp8:
                    i = s.inverse[0]
                    serving_plain.close(serving_plain.e4m3_values(got_k), (y * i).clamp(-448, 448), plain.in_e4m3(y * i, (bound + y.abs() * plain.U32) * i))
                    v8 = (v.float() * s.inverse[1]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
                    assert torch.equal(got_v, v8)
                else:
                    serving_plain.close(got_k, y, plain.in_half(y, bound))
                    assert torch.equal(got_v, v)
        tokens = int(s.starts[-1])
        want, bound = serving_plain.attention(s.q_out[:tokens], s.key[1], s.value[1], s.tables[at], s.starts, s.planned, -1, 0, s.d**-0.5,
                                              1 / s.inverse[0], 1 / s.inverse[1])
        serving_plain.close(s.o[:tokens], want, bound, "attention")
        s.score()
        before = s.tables[at].tolist()
        s.choose(at)
        found = plain.select(s.logits.cpu(), s.scores.cpu(), s.ended.cpu(), 7, s.beams)
        assert s.tokens.tolist() == found[1] and s.parents.tolist() == found[2] and s.new_ended.tolist() == found[3]
        assert int(s.info[2]) == 0
        forks += int(s.info[1])
        parents, chosen = s.parents.view(-1).tolist(), s.tokens.view(-1).tolist()
        adds, was = s.move()
        for r, (p, n) in enumerate(zip(parents, s.lengths[1 - at].tolist())):
            assert n == (len(histories[p]) if p >= 0 else 0)
            assert s.tables[1 - at][r, :n // s.page].tolist() == (before[p][:n // s.page] if p >= 0 else [])
        histories = [list(histories[p]) if p >= 0 else [] for p in parents]
        for r, h in enumerate(histories):
            assert [t for t in s.history.view(s.rows, -1)[r].tolist() if t >= 0][:len(h)] == h
            if bool(adds[r]):
                h.append(chosen[r])
                s.history.view(s.rows, -1)[r, len(h) - 1] = chosen[r]
        if not bool(adds.any()):
            break
        s.feed(torch.tensor([c for c, a in zip(chosen, adds.tolist()) if a], device="cuda"))
        # nothing is lost: the free pages and the listed ones are all
        begin, end = s.range.tolist()
        used = {p for row, n in zip(s.tables[1 - at].tolist(), s.lengths[1 - at].tolist()) for p in row[:-(-n // s.page)]}
        assert sorted(used | set(s.free.tolist()[begin:end])) == list(range(s.freed.numel())) and end - begin + len(used) == s.freed.numel()
    assert step >= 5 and forks > 4


def test_beam_search_in_graphs(pk):  # noqa: F811
    """Replayed halves of a step (one graph for each direction of the tables) equal eager ones bit for bit."""
    eager, graphed = Search(pk, False, 17), Search(pk, False, 17)
    graphs = []
    for at in (0, 1):
        both = []
        for half in (graphed.attend, graphed.choose):
            half(at)  # no token is asked for yet
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                half(at)
            both.append(graph)
        graphs.append(both)
    for name, t in vars(eager).items():
        for u, w in zip(t if isinstance(t, list) else [t], getattr(graphed, name) if isinstance(t, list) else [getattr(graphed, name)]):
            if torch.is_tensor(u) and not name.endswith("space"):
                w.copy_(u)
    gens = gen(5), gen(5)
    eager.begin(gens[0])
    graphed.begin(gens[1])
    for step in range(12):
        at = step % 2
        eager.attend(at)
        graphs[at][0].replay()
        for s in (eager, graphed):
            s.score()
        eager.choose(at)
        graphs[at][1].replay()
        torch.cuda.synchronize()
        bits = lambda t: t.view(torch.int16) if t.dtype is torch.float16 else t  # noqa: E731
        for a, b in zip(eager.outputs(), graphed.outputs()):
            assert torch.equal(bits(a), bits(b))
        for s in (eager, graphed):
            chosen = s.tokens.view(-1)
            adds, _ = s.move()
            s.feed(chosen[adds].long())
