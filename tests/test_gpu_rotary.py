"""Norm of query and key heads with the rotation by position, with and without the write into the paged cache."""
import math

import pytest

torch = pytest.importorskip("torch")

import decoding_plain as plain  # noqa: E402
import serving_plain  # noqa: E402
from serving_plain import close  # noqa: E402
from test_gpu_parity import pk  # noqa: E402, F401
from test_gpu_serving import gen, randn  # noqa: E402

pytestmark = pytest.mark.gpu


def ints(g, lo, hi, *shape):
    return torch.randint(lo, hi + 1, shape, generator=g, device="cuda", dtype=torch.int32)


class Heads:
    """Queries, keys and values as slices of one projection's rows."""

    def __init__(self, pk, tokens, heads, kv, d, r, seed=0, weights=True, far=1 << 20, scale=1.0):  # noqa: F811
        g = gen(seed + 7 * tokens + d + r)
        self.rows = randn(g, tokens, heads + 2 * kv, d, scale=scale)
        self.q, self.k, self.v = self.rows[:, :heads], self.rows[:, heads:heads + kv], self.rows[:, heads + kv:]
        self.qw, self.kw = (randn(g, d), randn(g, d)) if weights else (None, None)
        self.positions = ints(g, 0, far, tokens)
        self.words = pk.rotary_frequencies(r) if r else None
        self.q_out, self.k_out = (torch.full((tokens, n, d), 9.0, dtype=torch.float16, device="cuda") for n in (heads, kv))

    def check(self, interleaved, amplitude, eps, q_out=None, k_out=None, rows=None):
        rows = self.rows if rows is None else rows
        heads, kv = self.q.shape[1], self.k.shape[1]
        for x, w, got in ((rows[:, :heads], self.qw, self.q_out if q_out is None else q_out),
                          (rows[:, heads:heads + kv], self.kw, self.k_out if k_out is None else k_out)):
            y, bound = plain.head_norm_rotary(x, w, self.positions, self.words, interleaved, amplitude, eps)
            close(got, y, plain.in_half(y, bound))


@pytest.mark.parametrize("tokens,heads,kv,d,r", [
    (1, 8, 8, 128, 128), (1, 1, 1, 32, 16), (3, 5, 1, 64, 64), (7, 32, 8, 128, 64), (17, 3, 3, 80, 80), (5, 6, 2, 96, 32), (2, 40, 8, 128, 128),
    (33, 7, 1, 192, 48), (9, 4, 4, 256, 256), (300, 16, 2, 64, 32), (11, 2, 1, 48, 48), (4, 3, 1, 112, 16), (1025, 9, 3, 128, 128), (6, 8, 2, 128, 0)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("weights", [False, True])
def test_head_norm_rotary(pk, tokens, heads, kv, d, r, interleaved, weights):  # noqa: F811
    h = Heads(pk, tokens, heads, kv, d, r, weights=weights)
    pk.head_norm_rotary(h.q, h.k, h.qw, h.kw, h.positions, h.words, h.q_out, h.k_out, interleaved=interleaved, amplitude=1.25, epsilon=1e-5)
    h.check(interleaved, 1.25, 1e-5)


@pytest.mark.parametrize("tokens", [9000])
@pytest.mark.parametrize("d", [64, 128, 160])
def test_many_tokens(pk, tokens, d):  # noqa: F811
    """So many that a wave takes all heads of its token."""
    h = Heads(pk, tokens, 10, 3, d, 32, far=300)
    pk.head_norm_rotary(h.q, h.k, h.qw, None, h.positions, h.words, h.q_out, h.k_out)
    h.kw = None
    h.check(False, 1.0, 1e-6)


@pytest.mark.parametrize("interleaved", [False, True])
def test_far_and_negative_positions(pk, interleaved):  # noqa: F811
    h = Heads(pk, 12, 4, 2, 128, 128)
    h.positions.copy_(torch.tensor([0, 1, -1, 2**31 - 1, -2**31, 10**9, 1 << 24, (1 << 24) + 1, 123456789, -77, 2, 3], dtype=torch.int32))
    pk.head_norm_rotary(h.q, h.k, h.qw, h.kw, h.positions, h.words, h.q_out, h.k_out, interleaved=interleaved)
    h.check(interleaved, 1.0, 1e-6)


def test_quarter_turns(pk):  # noqa: F811
    """Frequencies that are exact parts of a turn: borders of the quarters, to the last bit of the phase."""
    h = Heads(pk, 64, 2, 1, 32, 32, weights=False)
    steps = [1 << 60, 1 << 61, 1 << 62, 3 << 61, (1 << 61) - 1, (1 << 61) + 1, 7 << 60, 5 << 61, 0, 1, (1 << 63) - 1, -(1 << 63), -1, -(1 << 61), 12345, 1 << 32]
    h.words = torch.tensor([s if s < 1 << 63 else s - (1 << 64) for s in steps], dtype=torch.int64, device="cuda")
    h.positions = torch.arange(64, dtype=torch.int32, device="cuda") - 20
    for interleaved in (False, True):
        pk.head_norm_rotary(h.q, h.k, None, None, h.positions, h.words, h.q_out, h.k_out, interleaved=interleaved)
        h.check(interleaved, 1.0, 1e-6)


@pytest.mark.parametrize("interleaved", [False, True])
def test_in_place_in_slices(pk, interleaved):  # noqa: F811
    h = Heads(pk, 21, 6, 2, 64, 32)
    before = h.rows.clone()
    pk.head_norm_rotary(h.q, h.k, h.qw, h.kw, h.positions, h.words, h.q, h.k, interleaved=interleaved)
    h.check(interleaved, 1.0, 1e-6, h.q, h.k, before)
    assert torch.equal(h.v, before[:, 8:])


def test_queries_alone_and_keys_of_another_array(pk):  # noqa: F811
    h = Heads(pk, 5, 6, 2, 64, 64)
    pk.head_norm_rotary(h.q, None, h.qw, None, h.positions, h.words, h.q_out, None)
    whole = h.q_out.clone()
    h.q_out.fill_(9)
    pk.head_norm_rotary(h.q, h.k.contiguous(), h.qw, h.kw, h.positions, h.words, h.q_out, h.k_out)
    assert torch.equal(whole, h.q_out)
    h.check(False, 1.0, 1e-6)


@pytest.mark.parametrize("eps", [0.0, 1e-6])
@pytest.mark.parametrize("interleaved", [False, True])
def test_zeros_infinities_and_nan_stay_in_their_heads(pk, eps, interleaved):  # noqa: F811
    h = Heads(pk, 6, 8, 2, 128, 64)
    h.rows[0, 1] = 0
    h.rows[1, 0, 3] = math.inf    # normed: NaN there, zeros elsewhere in the head
    h.rows[2, 7, 100] = math.nan
    h.rows[3, 8, 90] = -math.inf  # a key, outside of the rotation
    h.rows[4, 2] = 6e4
    pk.head_norm_rotary(h.q, h.k, h.qw, h.kw, h.positions, h.words, h.q_out, h.k_out, interleaved=interleaved, epsilon=eps)
    for i, (t, head) in enumerate([(1, 0), (2, 7), (3, 8)]):
        got = (h.q_out if head < 8 else h.k_out)[t, head % 8].float()
        assert torch.isnan(got).any()
        if i == 2:  # an infinity alone in its head's norm: NaN at its place, the rest 0
            assert torch.isnan(got[90]) and not got[torch.arange(128, device="cuda") != 90].any()
    bad = torch.zeros(6, 10, dtype=torch.bool, device="cuda")
    bad[1, 0] = bad[2, 7] = bad[3, 8] = True
    for x, w, got, odd in ((h.q, h.qw, h.q_out, bad[:, :8]), (h.k, h.kw, h.k_out, bad[:, 8:])):
        y, bound = plain.head_norm_rotary(x, w, h.positions, h.words, interleaved, 1.0, eps)
        close(got[~odd], y[~odd], plain.in_half(y, bound)[~odd])
    assert not h.q_out[0, 1].any()


def test_infinity_without_norm_outside_of_the_rotation(pk):  # noqa: F811
    h = Heads(pk, 1, 1, 1, 64, 32, weights=False)
    h.rows[0, 0, 40] = math.inf
    pk.head_norm_rotary(h.q, h.k, None, None, h.positions, h.words, h.q_out, h.k_out)
    h.check(False, 1.0, 1e-6)


# ---- with the write into the cache --------------------------------------------------------

def make_cache(pages, kv, page, d, fp8):
    kind = torch.uint8 if fp8 else torch.float16
    return (torch.full((pages, kv, page, d), 3, dtype=kind, device="cuda"), torch.full((pages, kv, d, page), 3, dtype=kind, device="cuda"))


def slots_for(g, tokens, page, pages, how):
    if how == "runs":  # prompts: tokens of a page follow each other
        n = -(-tokens // page)
        ids = torch.randperm(pages, generator=g, device="cuda")[:n + 1]
        at = torch.arange(tokens, device="cuda") + 5
        return (ids[at // page] * page + at % page).int()
    return torch.randperm(pages * page, generator=g, device="cuda")[:tokens].int()


@pytest.mark.parametrize("tokens,heads,kv,d,r,page,how", [
    (1, 8, 8, 128, 128, 16, "scattered"), (5, 4, 2, 64, 32, 16, "scattered"), (61, 32, 8, 128, 64, 64, "scattered"), (200, 6, 3, 64, 64, 256, "runs"),
    (767, 4, 2, 128, 128, 32, "runs"), (768, 4, 2, 128, 128, 32, "runs"), (800, 3, 2, 64, 32, 16, "scattered"), (1535, 4, 2, 128, 128, 32, "runs"), (1536, 4, 2, 128, 128, 32, "runs"), (1700, 5, 1, 64, 48, 16, "scattered"), (2500, 4, 4, 64, 64, 128, "runs"),
    (3001, 3, 1, 128, 0, 64, "runs"), (9001, 4, 2, 64, 64, 64, "runs")])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
def test_write(pk, tokens, heads, kv, d, r, page, how, fp8, interleaved):  # noqa: F811
    h = Heads(pk, tokens, heads, kv, d, r, far=5000)
    g = gen(tokens)
    pages = 2 * (-(-tokens // page)) + 3
    slots = slots_for(g, tokens, page, pages, how)
    skip = torch.rand(tokens, generator=g, device="cuda") < 0.1
    skip[0] = False
    skip[-3:] = tokens > 4
    slots[skip] = torch.where(torch.arange(int(skip.sum()), device="cuda") % 2 == 0, -1, pages * page).int()
    key, value = make_cache(pages, kv, page, d, fp8)
    ki, vi = (4.0, 3.0) if fp8 else (1.0, 1.0)
    pk.head_norm_rotary_write(h.q, h.k, h.v, h.qw, h.kw, h.positions, slots, h.words, h.q_out, key, value, ki, vi, interleaved=interleaved, amplitude=0.75,
                              epsilon=1e-5)
    y, bound = plain.head_norm_rotary(h.q, h.qw, h.positions, h.words, interleaved, 0.75, 1e-5)
    close(h.q_out[~skip], y[~skip], plain.in_half(y, bound)[~skip])
    assert (h.q_out[skip] == 9).all()
    at = slots[~skip].long()
    y, bound = plain.head_norm_rotary(h.k, h.kw, h.positions, h.words, interleaved, 0.75, 1e-5)
    y, bound = y[~skip] * ki, bound[~skip] * ki
    got = key[at // page, :, at % page]
    if fp8:
        close(serving_plain.e4m3_values(got), y.clamp(-448, 448), plain.in_e4m3(y, bound + y.abs() * plain.U32))
        v = (h.v.float() * vi).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        close(got, y, plain.in_half(y, bound))
        v = h.v
    assert torch.equal(value.transpose(2, 3)[at // page, :, at % page], v[~skip])
    untouched = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    untouched[at] = False
    u = untouched.nonzero()[:, 0]
    assert (key[u // page, :, u % page] == 3).all() and (value.transpose(2, 3)[u // page, :, u % page] == 3).all()


@pytest.mark.parametrize("tokens", [40, 2000])
def test_write_in_fp16_equals_the_two_calls(pk, tokens):  # noqa: F811
    h = Heads(pk, tokens, 8, 2, 128, 128)
    slots = slots_for(gen(1), tokens, 64, 80, "runs")
    caches = [make_cache(80, 2, 64, 128, False) for _ in range(2)]
    pk.head_norm_rotary_write(h.q, h.k, h.v, h.qw, h.kw, h.positions, slots, h.words, h.q_out, *caches[0])
    one = h.q_out.clone()
    pk.head_norm_rotary(h.q, h.k, h.qw, h.kw, h.positions, h.words, h.q_out, h.k_out)
    pk.paged_cache_write(h.k_out, h.v, slots, *caches[1])
    assert torch.equal(one, h.q_out)
    for a, b in zip(*caches):
        assert torch.equal(a, b)


def test_write_queries_in_place(pk):  # noqa: F811
    h = Heads(pk, 30, 8, 2, 64, 64)
    before = h.rows.clone()
    slots = slots_for(gen(1), 30, 16, 8, "scattered")
    key, value = make_cache(8, 2, 16, 64, True)
    pk.head_norm_rotary_write(h.q, h.k, h.v, h.qw, h.kw, h.positions, slots, h.words, h.q, key, value)
    y, bound = plain.head_norm_rotary(before[:, :8], h.qw, h.positions, h.words, False, 1.0, 1e-6)
    close(h.q, y, plain.in_half(y, bound))
    assert torch.equal(h.rows[:, 8:], before[:, 8:])


@pytest.mark.parametrize("tokens", [3, 1600])
@pytest.mark.parametrize("fp8", [False, True])
def test_write_beyond_32_bit_offsets(pk, tokens, fp8):  # noqa: F811
    kv, d, page = 8, 128, 256
    pages = (1 << 32) // (kv * d * page) + 40
    kind = torch.uint8 if fp8 else torch.float16
    key = torch.empty((pages, kv, page, d), dtype=kind, device="cuda")
    value = torch.empty((pages, kv, d, page), dtype=kind, device="cuda")
    h = Heads(pk, tokens, 4, kv, d, 64)
    at = torch.arange(tokens, device="cuda") + 7
    slots = ((pages - 1 - at // page) * page + at % page).int()
    pk.head_norm_rotary_write(h.q, h.k, h.v, h.qw, h.kw, h.positions, slots, h.words, h.q_out, key, value)
    y, bound = plain.head_norm_rotary(h.k, h.kw, h.positions, h.words, False, 1.0, 1e-6)
    s = slots.long()
    got = key[s // page, :, s % page]
    if fp8:
        close(serving_plain.e4m3_values(got), y, plain.in_e4m3(y, bound + y.abs() * plain.U32))
    else:
        close(got, y, plain.in_half(y, bound))
    v = h.v.float().to(torch.float8_e4m3fn).view(torch.uint8) if fp8 else h.v
    for i in (0, 1, tokens - 1):
        assert torch.equal(value[int(s[i]) // page, :, :, int(s[i]) % page], v[i])


def test_e4m3_keys_saturate_and_keep_nan(pk):  # noqa: F811
    h = Heads(pk, 2, 2, 1, 64, 32, weights=False)
    h.rows[0, 2, 50] = 1000
    h.rows[0, 2, 51] = math.nan
    h.rows[1, 2, 52] = -math.inf
    key, value = make_cache(1, 1, 16, 64, True)
    pk.head_norm_rotary_write(h.q, h.k, h.v, None, None, h.positions, torch.tensor([2, 3], dtype=torch.int32, device="cuda"), h.words, h.q_out, key, value)
    assert key[0, 0, 2, 50] == 0x7E and key[0, 0, 2, 51] & 0x7F == 0x7F and key[0, 0, 3, 52] == 0xFE


@pytest.mark.parametrize("tokens", [1, 50, 1600])
def test_replays_follow_positions_and_slots(pk, tokens):  # noqa: F811
    h = Heads(pk, tokens, 8, 2, 64, 64)
    key, value = make_cache(120, 2, 16, 64, False)
    want = [torch.full_like(key, 3), torch.full_like(value, 3)]
    g = gen(2)
    slots = torch.full((tokens,), -1, dtype=torch.int32, device="cuda")
    call = lambda out, caches: pk.head_norm_rotary_write(h.q, h.k, h.v, h.qw, h.kw, h.positions, slots, h.words, out, *caches)  # noqa: E731
    call(h.q_out, (key, value))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(h.q_out, (key, value))
    for _ in range(4):
        h.rows.copy_(randn(g, *h.rows.shape))
        h.positions.copy_(ints(g, 0, 10000, tokens))
        slots.copy_(slots_for(g, tokens, 16, 120, "scattered"))
        graph.replay()
        out = torch.full_like(h.q_out, 9)
        call(out, want)
        torch.cuda.synchronize()
        assert torch.equal(out, h.q_out) and torch.equal(key, want[0]) and torch.equal(value, want[1])


def test_on_two_streams_at_once(pk):  # noqa: F811
    sets = [Heads(pk, 500, 8, 2, 128, 128, seed=s) for s in (1, 2)]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for h, s in zip(sets, streams):
        with torch.cuda.stream(s):
            torch.cuda._sleep(200000)
        pk.head_norm_rotary(h.q, h.k, h.qw, h.kw, h.positions, h.words, h.q_out, h.k_out, stream=s)
    torch.cuda.synchronize()
    for h in sets:
        h.check(False, 1.0, 1e-6)
