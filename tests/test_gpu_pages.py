"""Pages that follow their beams: forks of block tables, the free list, copies of pages."""
import random

import pytest

torch = pytest.importorskip("torch")

import decoding_plain as plain  # noqa: E402
import serving_plain  # noqa: E402
from test_gpu_parity import pk  # noqa: E402, F401
from test_gpu_serving import gen, randn  # noqa: E402

pytestmark = pytest.mark.gpu


def dev(x, kind=torch.int32):
    return torch.tensor(x, dtype=kind, device="cuda")


class Pool:
    """Tables of a few rows over pages that rows may share, and a free list, in lists and on the GPU."""

    def __init__(self, rng, rows, columns, page, spare=50, groups=1):
        self.page, self.rows, self.columns = page, rows, columns
        ids = list(range(rows * columns + spare))
        rng.shuffle(ids)
        self.pages = len(ids)
        self.table, self.lengths = [], []
        for r in range(rows):
            n = rng.choice([0, 1, page, rng.randint(0, columns * page), rng.randint(0, columns * page), columns * page])
            need = -(-n // page)
            row = []
            if self.table and rng.random() < 0.7:  # full pages of another row in front
                other = rng.randrange(r)
                row = self.table[other][:min(rng.randint(0, columns), self.lengths[other] // page, n // page)]
            row = row + [ids.pop() for _ in range(need - len(row))]
            self.table.append(row + [-7] * (columns - need))
            self.lengths.append(n)
        self.begin = rng.randint(0, 3)
        self.free = [-5] * self.begin + ids
        self.end = len(self.free)

    def run(self, pk, parents, held=None, workspace=None, end=None):  # noqa: F811
        self.range = dev([self.begin, self.end if end is None else end])
        self.new_table, self.new_lengths = dev([[-3] * self.columns] * self.rows), dev([-3] * self.rows)
        self.copies, self.freed, self.info = dev([[-3, -3]] * self.rows), torch.full((self.pages,), -3, dtype=torch.int32, device="cuda"), dev([9] * 4)
        size = pk.page_fork_workspace_bytes(self.rows, self.columns, self.pages)
        workspace = torch.full((size,), 0xFF, dtype=torch.uint8, device="cuda") if workspace is None else workspace
        given = [dev(parents), dev(self.table), dev(self.lengths), dev(self.free)]
        before = [t.clone() for t in given]
        pk.page_fork(*given, self.range, self.new_table, self.new_lengths, self.copies, self.freed, self.info, workspace, self.page,
                     None if held is None else dev(held, torch.uint8))
        for t, u in zip(given, before):
            assert torch.equal(t, u)

    def check(self, parents, held=None, end=None):
        want = plain.fork(parents, self.table, self.lengths, self.free, self.begin, self.end if end is None else end, self.page, self.pages, held)
        assert self.info.tolist() == want[4]
        assert self.new_lengths.tolist() == want[1]
        assert self.new_table.tolist() == [row + [-3] * (self.columns - len(row)) for row in want[0]]
        assert self.copies.tolist() == want[2]
        assert self.freed.tolist() == want[3] + [-3] * (self.pages - len(want[3]))
        assert self.range.tolist()[0] == self.begin
        return want

    def go(self, pk, parents, held=None, end=None):  # noqa: F811
        self.run(pk, parents, held, end=end)
        return self.check(parents, held, end)


@pytest.mark.parametrize("rows,columns,page", [(1, 1, 16), (2, 3, 16), (4, 5, 32), (16, 29, 16), (33, 8, 256), (100, 70, 64), (1025, 3, 128), (4096, 5, 16)])
@pytest.mark.parametrize("seed", [0, 1, 2])
def test_fork(pk, rows, columns, page, seed):  # noqa: F811
    rng = random.Random(rows + seed)
    pool = Pool(rng, rows, columns, page, spare=rows + 20)
    pool.go(pk, list(range(rows)))  # nothing changes
    pool.go(pk, [-1] * rows)        # all go back
    pool.go(pk, [rng.randrange(rows)] * rows)
    for _ in range(3):
        parents = [-1 if rng.random() < 0.2 else rng.randrange(rows) for _ in range(rows)]
        held = [int(rng.random() < 0.3) for _ in range(pool.pages)]
        pool.go(pk, parents)
        pool.go(pk, parents, held)


def test_fork_refuses_all_or_nothing(pk):  # noqa: F811
    rng = random.Random(4)
    pool = Pool(rng, 6, 4, 16)
    pool.lengths = [17, 5, 33, 64, 0, 3]
    pool.table = [[r * 4 + c if c < -(-n // 16) else -7 for c in range(4)] for r, n in enumerate(pool.lengths)]
    assert pool.go(pk, [0, 0, 0, 1, 1, 4], end=pool.begin + 2)[4] == [0, 0, 1, 0]  # three pages needed
    assert pool.go(pk, [0, 0, 0, 1, 1, 4], end=pool.begin + 3)[4][:3] == [6, 3, 0]
    assert pool.go(pk, [0, 0, 0, 1, 1, 4], end=pool.end + 1000)[4][:3] == [6, 3, 0]  # no further than the list
    assert pool.go(pk, [3, 3, 3, 3, -1, -1], end=pool.begin - 2)[4] == [4, 0, 0, 7]  # full pages: none is needed
    for bad in ([0, 1, 2, 3, 4, 6], [0, -2, 2, 3, 4, 5], [2**31 - 1] + [0] * 5, [-2**31] + [0] * 5):
        assert pool.go(pk, bad)[4] == [0, 0, 8, 0]
    for bad in (-1, 65, 2**31 - 1, -2**31):
        pool.lengths[5] = bad
        assert pool.go(pk, [0, 0, 1, 1, 2, 2])[4] == [0, 0, 8, 0]
    pool.lengths[5], pool.begin = 3, -1
    assert pool.go(pk, [0, 0, 1, 1, 2, 2])[4] == [0, 0, 8, 0]


def test_fork_passes_odd_pages_on(pk):  # noqa: F811
    pool = Pool(random.Random(1), 4, 3, 16, spare=20)
    pool.lengths = [40, 40, 20, 0]
    pool.table = [[-1, 2, 3], [4, pool.pages, 2**31 - 1], [5, -2**31, -7], [-7] * 3]
    want = pool.go(pk, [0, 0, 1, 1])
    assert want[4] == [4, 1, 0, 1] and want[3] == [5]
    pool.go(pk, [2, 2, -1, -1])


@pytest.mark.parametrize("pages", [4095, 4096, 4097, 70001, (1 << 22) + 3])
def test_fork_of_large_pools(pk, pages):  # noqa: F811
    """Pages that go back at the ends of a pool and of the parts that workgroups list."""
    rows, columns, page = 3, 40, 16
    pool = Pool(random.Random(2), rows, columns, page)
    pool.pages = pages
    edge = [0, 1, 15, 16, 4079, 4094, pages - 1, pages - 2, pages // 2] + ([4096, 8191, 8192, 65535, 65536] if pages > 70000 else [])
    pool.table = [[edge[c % len(edge)] for c in range(columns)], [200 + c for c in range(columns)], [200 + c if c < 7 else 300 + c for c in range(columns)]]
    pool.lengths = [16 * len(edge), 640, 631]
    pool.free, pool.begin, pool.end = [9, 10, 11, 12], 0, 4
    pool.go(pk, [2, 2, -1])
    pool.go(pk, [1, -1, 1])
    pool.go(pk, [-1, -1, -1])


@pytest.mark.parametrize("pages", [(1 << 17) + 1, 200003, (1 << 21) - 31, 1 << 21, (1 << 21) + 1])
def test_fork_of_pools_listed_by_several_workgroups(pk, pages):  # noqa: F811
    rng = random.Random(pages)
    rows, columns, page = 24, 90, 32
    pool = Pool(rng, rows, columns, page)
    some = sorted({0, 31, 32, 127, 32767, 32768, 65535, 65536, 98304, pages - 1, pages - 2} | set(rng.sample(range(pages), rows * columns)))
    ids = some[:11] + some[-11:] + some[11:-11]
    pool.table = [[ids[(r * columns + c) % len(ids)] if c < -(-n // page) else -7 for c in range(columns)] for r, n in enumerate(pool.lengths)]
    pool.free, pool.begin, pool.end, pool.pages = [i for i in range(50000, 50100)], 2, 100, pages
    pool.go(pk, [-1] * rows)
    for _ in range(2):
        parents = [-1 if rng.random() < 0.3 else rng.randrange(rows) for _ in range(rows)]
        pool.go(pk, parents)
        held = bytearray(pages)
        for i in rng.sample(ids, len(ids) // 3):
            held[i] = 1 + i % 255
        pool.go(pk, parents, list(held))


def test_fork_with_a_larger_workspace_and_replays(pk):  # noqa: F811
    rng = random.Random(8)
    pool = Pool(rng, 12, 9, 16)
    space = torch.full((pk.page_fork_workspace_bytes(40, 30, 5000),), 0xFF, dtype=torch.uint8, device="cuda")
    parents = [0, 0, 1, 1, 1, -1, 7, 8, 9, 9, 3, 3]
    pool.run(pk, parents, workspace=space)
    pool.check(parents)
    given = [dev(parents), dev(pool.table), dev(pool.lengths), dev(pool.free), pool.range]
    call = lambda: pk.page_fork(*given, pool.new_table, pool.new_lengths, pool.copies, pool.freed, pool.info, space, 16)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for _ in range(4):
        parents = [rng.randrange(-1, 12) for _ in range(12)]
        given[0].copy_(dev(parents))
        for t in (pool.new_table, pool.copies, pool.freed, space.view(torch.int32) if space.numel() % 4 == 0 else pool.info):
            t.fill_(-3)
        graph.replay()
        torch.cuda.synchronize()
        pool.check(parents)


def test_fork_of_a_large_table_replays(pk):  # noqa: F811
    """The several launches of one call, and two calls that share a workspace one behind the other."""
    rng = random.Random(21)
    pools = [Pool(rng, rows, 7, 16, spare=rows) for rows in (1100, 1300)]
    space = torch.full((pk.page_fork_workspace_bytes(1300, 7, max(p.pages for p in pools)),), 0xFF, dtype=torch.uint8, device="cuda")
    parents, given = [], []
    for p in pools:
        ids = [rng.randrange(-1, p.rows) for _ in range(p.rows)]
        p.run(pk, ids, workspace=space)
        p.check(ids)
        given.append([dev(ids), dev(p.table), dev(p.lengths), dev(p.free), p.range])
    call = lambda: [pk.page_fork(*g, p.new_table, p.new_lengths, p.copies, p.freed, p.info, space, p.page) for g, p in zip(given, pools)]  # noqa: E731
    graph = torch.cuda.CUDAGraph()
    call()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        call()
    for _ in range(3):
        parents = [[rng.randrange(-1, p.rows) for _ in range(p.rows)] for p in pools]
        for g, p, ids in zip(given, pools, parents):
            g[0].copy_(dev(ids))
            for t in (p.new_table, p.copies, p.freed):
                t.fill_(-3)
        space.fill_(0xFF)
        graph.replay()
        torch.cuda.synchronize()
        for p, ids in zip(pools, parents):
            p.check(ids)


def test_keep(pk):  # noqa: F811
    free, freed = dev(list(range(100, 140))), dev([7, 8, 9, 50, 51])
    run = lambda info, begin, freed=freed: (  # noqa: E731
        lambda f, r: (pk.page_keep(dev(info), freed, f, r), f.tolist(), r.tolist())[1:])(free.clone(), dev([begin, 30]))
    base = list(range(100, 140))
    assert run([0, 4, 0, 0], 10) == (base, [14, 30])
    assert run([0, 4, 0, 3], 10, None) == (base, [14, 30])
    assert run([0, 4, 2, 3], 10) == (base, [10, 30])
    assert run([0, 1, 0, 3], 10) == (base[:8] + [7, 8, 9] + base[11:], [8, 30])
    assert run([0, 5, 0, 5], 0) == ([7, 8, 9, 50, 51] + base[5:], [0, 30])
    assert run([0, 1, 0, 5], 1) == ([7, 8] + base[2:], [0, 30])  # room for two
    assert run([0, 1, 0, 9], 10) == (base[:6] + [7, 8, 9, 50, 51] + base[11:], [6, 30])  # more than freed holds
    assert run([0, 1, 0, -2], 10) == (base, [11, 30])
    assert run([0, 1, 0, 3], 10, freed[:0]) == (base, [11, 30])


def test_keep_many(pk):  # noqa: F811
    n = 100000
    free, freed, r = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.arange(n, dtype=torch.int32, device="cuda"), dev([n - 1, n])
    pk.page_keep(dev([0, 1, 0, n - 5]), freed, free, r)
    assert r.tolist() == [5, n] and torch.equal(free[5:], freed[:n - 5]) and not free[:5].any()


@pytest.mark.parametrize("pages,kv,page,d,layers", [(7, 1, 16, 64, 1), (9, 3, 16, 64, 2), (40, 8, 64, 128, 1), (12, 2, 256, 128, 5), (30, 8, 16, 128, 24)])
@pytest.mark.parametrize("fp8", [False, True])
def test_copy(pk, pages, kv, page, d, layers, fp8):  # noqa: F811
    g = gen(pages)
    shape = (pages,) if layers == 1 else (layers, pages)
    make = lambda *s: torch.randint(0, 200, shape + s, generator=g, device="cuda", dtype=torch.uint8) if fp8 else randn(g, *shape, *s)  # noqa: E731
    key, value = make(kv, page, d), make(kv, d, page)
    ids = torch.randperm(pages, generator=g, device="cuda").tolist()
    half = pages // 2
    pairs = [[s, t] for s, t in zip(ids[:half], ids[half:2 * half])]
    pairs[0][0] = pairs[1][0]  # a page that two take
    pairs += [[-1, -1], [pages, 1], [1, pages], [-1, 0], [0, -5], [2**31 - 1, 0], [ids[0], ids[0]]]
    want = [key.clone(), value.clone()]
    for s, t in pairs[:half]:
        for x in want:
            if layers == 1:
                x[t] = x[s]
            else:
                x[:, t] = x[:, s]
    pk.paged_cache_copy(dev(pairs), key, value)
    assert torch.equal(key, want[0]) and torch.equal(value, want[1])


def test_copy_beyond_32_bits(pk):  # noqa: F811
    kv, d, page = 8, 128, 256
    pages = (1 << 32) // (kv * d * page) + 40
    key, value = torch.empty((pages, kv, page, d), dtype=torch.float16, device="cuda"), torch.empty((pages, kv, d, page), dtype=torch.float16, device="cuda")
    g = gen(1)
    key[3], value[3], key[pages - 1], value[pages - 1] = (randn(g, kv, a, b) for a, b in ((page, d), (d, page), (page, d), (d, page)))
    pk.paged_cache_copy(dev([[3, pages - 2], [pages - 1, 5], [-1, -1]]), key, value)
    for x in (key, value):
        assert torch.equal(x[pages - 2], x[3]) and torch.equal(x[5], x[pages - 1])


def test_free_list_through_plans_and_forks(pk):  # noqa: F811
    """Many steps of plan, fork and keep: no page is lost, none is listed twice but for shared full ones."""
    rng = random.Random(11)
    rows, columns, page = 8, 12, 16
    pages = 70
    free, free_range = dev(rng.sample(range(pages), pages)), dev([0, pages])
    tables, lengths = [dev([[-1] * columns] * rows) for _ in range(2)], [dev([0] * rows) for _ in range(2)]
    added, starts, slots, positions = dev([0] * rows), dev([0] * (rows + 1)), dev([0] * 64), dev([0] * 64)
    plan_info, info, copies, freed, planned = dev([0] * 4), dev([0] * 4), dev([[0, 0]] * rows), dev([0] * pages), dev([0] * rows)
    space = torch.empty(pk.page_fork_workspace_bytes(rows, columns, pages), dtype=torch.uint8, device="cuda")
    forked = refused = 0
    for step in range(60):
        a, b = step % 2, 1 - step % 2
        held = lengths[a].tolist()
        added.copy_(dev([rng.randint(0, 7) if n < columns * page - 7 else 0 for n in held]))
        pk.page_plan(lengths[a], added, free, free_range, tables[a], starts, planned, slots, positions, plan_info, page)
        pk.page_keep(plan_info, None, free, free_range)
        lengths[a].copy_(planned)
        parents = [-1 if rng.random() < 0.08 else rng.randrange(max(0, r - 2), min(rows, r + 2)) for r in range(rows)]
        before, now = tables[a].tolist(), lengths[a].tolist()
        begin, end = free_range.tolist()
        listing = free.tolist()
        tables[b].fill_(-1)
        pk.page_fork(dev(parents), tables[a], lengths[a], free, free_range, tables[b], lengths[b], copies, freed, info, space, page)
        want = plain.fork(parents, before, now, listing, begin, end, page, pages)
        assert info.tolist() == want[4] and lengths[b].tolist() == want[1] and copies.tolist() == want[2]
        assert [row[:-(-n // page)] for row, n in zip(tables[b].tolist(), want[1])] == want[0]
        forked, refused = forked + want[4][1], refused + (want[4][2] + plan_info.tolist()[2] > 0)
        pk.page_keep(info, freed, free, free_range)
        begin, end = free_range.tolist()
        left = free.tolist()[begin:end]
        used = [p for row, n in zip(tables[b].tolist(), lengths[b].tolist()) for p in row[:-(-n // page)]]
        last = [row[n // page] for row, n in zip(tables[b].tolist(), lengths[b].tolist()) if n % page]
        assert sorted(set(used) | set(left)) == list(range(pages)) and len(left) + len(set(used)) == pages
        assert all(used.count(p) == 1 for p in last)
    assert forked > 20
