"""Attention over the paged 8-bit cache against the 64-bit oracle.

Tolerances, derived: O is rounded once to bf16 (2^-8 of itself), and each
probability, times its page's scale, once (2^-8 of it, so at most 2^-8 of
sum_j p_j |v_j| together).  The rest is fp32: a score adds D products
(N(0, 1) values: sum |q k| / sqrt(D) stays under 20 here, so under
132 * 2^-24 * 20 = 2^-12.6, of which every probability is off by the same
part), then exp2, the sums and the joins of at most a few hundred terms:
2^-12 of sum_j p_j |v_j| in all, and 2^-12 absolute for the LSE."""
import math

import pytest
import torch

from oracle.layer_ref import attention_cached_ref, cache_write_ref
from oracle.torch_ref import seeded_normal
from tests.conftest import announce
from warpir_amd import api, kvcache

pytestmark = pytest.mark.gpu


def _ints(x):
    return torch.tensor(x, dtype=torch.int32)


def _cache(b, heads, page, d, columns, lengths, seed=0, spare=2):
    """(cache on the CPU, table) holding N(0, 1) keys and values of these lengths, pages in any order."""
    pages = b * columns + spare
    cache = api.KVCache.empty(pages, heads, page, d, device="cpu")
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))[:b * columns].view(b, columns).int()
    n = min(max(max(lengths), 1), columns * page)
    x = [seeded_normal((b, heads, n, d), seed + 1 + i, 1.0 + i) for i in range(2)]
    cache_write_ref(cache, *x, table, _ints([n] * b))
    for i, length in enumerate(lengths):   # pages past the end are no sequence's
        table[i, -(-min(max(length, 0), columns * page) // page):] = -1
    return cache, table


def _gpu(cache):
    return api.KVCache(*(x.cuda() for x in cache))


def _compare(got, q, cache, table, lengths, counts=None):
    o, lse, weight = attention_cached_ref(q.cpu(), cache, table, lengths, counts)
    off = (got[0].cpu().double() - o).abs()
    assert bool((off <= 2 ** -8 * o.abs() + (2 ** -8 + 2 ** -12) * weight).all()), off.max()
    empty = lse == -math.inf
    assert torch.equal(got[1].cpu() == -math.inf, empty)
    assert not bool((~empty).any()) or (got[1].cpu().double() - lse)[~empty].abs().max() <= 2 ** -12
    assert bool((got[0].cpu()[empty] == 0).all())


def _run(q, cache, table, lengths, counts=None, **more):
    return api.attention_cached(q.cuda(), cache, table.cuda(), _ints(lengths).cuda(),
                                counts=None if counts is None else _ints(counts).cuda(), **more)


CASES = [   # heads, kv heads, tokens, page, columns, lengths, counts
    (1, 1, 1, 16, 1, (1,), None),
    (4, 2, 1, 16, 40, (1, 15, 16, 17, 63, 64, 65, 0, 640, 127), None),
    (16, 1, 1, 64, 12, (700, 0, 768), None),
    (17, 1, 1, 32, 9, (288, 31), None),
    (8, 4, 3, 32, 20, (2, 5, 640, 3, 64), (2, 0, 3, 1, 3)),
    (8, 2, 4, 128, 5, (4, 640, 130), None),
    (8, 1, 5, 16, 24, (384, 100, 5), (5, 2, 5)),
    (6, 2, 29, 64, 6, (29, 384, 200), (29, 7, 12)),
    (4, 1, 70, 16, 30, (70, 480, 69), None),
    (2, 2, 300, 64, 8, (300, 511), (300, 150)),
    (3, 3, 129, 128, 4, (129, 500), None),
]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,hkv,tokens,page,columns,lengths,counts", CASES)
def test_against_the_oracle(gpu, heads, hkv, tokens, page, columns, lengths, counts, d):
    announce(f"attention cached H{heads}/{hkv} T{tokens} page {page} D{d} lengths {lengths} counts {counts}")
    cache, table = _cache(len(lengths), hkv, page, d, columns, lengths)
    q = seeded_normal((len(lengths), heads, tokens, d), 9)
    for _ in range(2):   # the call and its plan
        _compare(_run(q, _gpu(cache), table, lengths, counts), q, cache, table, lengths, counts)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,hkv,tokens", [(2, 1, 1), (20, 1, 1), (4, 1, 40)])
def test_long_sequences_in_many_parts(gpu, heads, hkv, tokens, d):
    """A head's keys over many programs, next to short ones; the same bits every time."""
    lengths = (9000, 70, 64, 5001)
    announce(f"attention cached long H{heads} T{tokens} D{d}")
    cache, table = _cache(4, hkv, 64, d, 150, lengths)
    q = seeded_normal((4, heads, tokens, d), 9)
    got = _run(q, _gpu(cache), table, lengths)
    _compare(got, q, cache, table, lengths)
    again = _run(q, _gpu(cache), table, lengths)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


@pytest.mark.parametrize("forced", [(16, 4, 7, 1), (16, 8, 3, 2), (128, 4, 5, 1), (32, 4, 512, 1), (128, 4, 0, 0),
                                    (16, 8, 0, 0), (16, 2, 0, 0), (32, 2, 0, 0), (16, 4, 1, 1), (32, 8, 70, 1), (128, 4, 512, 2), (16, 4, 13, 9)])
def test_every_division_gives_the_same(gpu, monkeypatch, forced):
    """Few programs that each take several heads' tiles, shares that end inside them, and no division."""
    lengths, counts = (130, 0, 400, 65), (3, 0, 3, 1)
    cache, table = _cache(4, 3, 16, 64, 26, lengths)
    q = seeded_normal((4, 9, 3, 64), 5)
    monkeypatch.setattr(kvcache, "_attention_form", lambda *a: forced)
    monkeypatch.setattr(kvcache, "_attention_plans", kvcache.DevicePlans("attention_cached"))
    _compare(_run(q, _gpu(cache), table, lengths, counts), q, cache, table, lengths, counts)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("forced", [(16, 4, 256, 2), (128, 8, 0, 0), (32, 4, 40, 1), (128, 4, 300, 2), (16, 4, 3, 1), (32, 4, 0, 0)])
def test_every_division_of_many_blocks(gpu, monkeypatch, forced, d):
    """Blocks that end inside a token's heads, some with nothing to see."""
    lengths, counts = (700, 0, 90, 300), (50, 0, 7, 33)
    cache, table = _cache(4, 2, 32, d, 23, lengths)
    q = seeded_normal((4, 6, 50, d), 5)
    monkeypatch.setattr(kvcache, "_attention_form", lambda *a: forced)
    monkeypatch.setattr(kvcache, "_attention_plans", kvcache.DevicePlans("attention_cached"))
    _compare(_run(q, _gpu(cache), table, lengths, counts), q, cache, table, lengths, counts)


@pytest.mark.parametrize("batch,heads,hkv,tokens,form", [
    (12, 32, 8, 256, (128, 4, 0, 0)), (1, 8, 1, 600, (128, 4, 0, 0)), (1, 4, 2, 333, (16, 4, 0, 0)),
    (3, 6, 3, 500, (128, 4, 0, 0)), (3, 6, 3, 500, (128, 8, 0, 0)), (4, 8, 4, 300, (128, 4, 0, 0)), (40, 8, 8, 300, (32, 4, 0, 0))])
def test_the_order_of_many_blocks(gpu, monkeypatch, batch, heads, hkv, tokens, form):
    """Every block is computed once, whatever the order: long before short, halves that turn round, by length."""
    lengths = [tokens + 13 * (i % 5) for i in range(batch)]
    cache, table = _cache(batch, hkv, 64, 64, 11, lengths)
    q = seeded_normal((batch, heads, tokens, 64), 5)
    monkeypatch.setattr(kvcache, "_attention_form", lambda *a: form)
    monkeypatch.setattr(kvcache, "_attention_plans", kvcache.DevicePlans("attention_cached"))
    _compare(_run(q, _gpu(cache), table, lengths), q, cache, table, lengths)


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("d", [64, 128])
def test_blocks_of_128_rows(gpu, monkeypatch, d, page):
    """Against the oracle with pages that are none, and where NaN codes and scales lie: as blocks of 16 rows have it."""
    lengths, counts = (700, 0, 90, 300), (50, 0, 7, 33)
    columns = -(-704 // page) + 1
    cache, table = _cache(4, 2, page, d, columns, lengths)
    q = seeded_normal((4, 6, 50, d), 5)

    def both(cache, table):
        got = []
        for form in ((128, 4, 0, 0), (16, 4, 0, 0), (128, 4, 300, 2), (128, 8, 0, 0)):
            monkeypatch.setattr(kvcache, "_attention_form", lambda *a: form)
            monkeypatch.setattr(kvcache, "_attention_plans", kvcache.DevicePlans("attention_cached"))
            got.append([x.cpu() for x in _run(q, _gpu(cache), table, lengths, counts)])
        return got

    holes = table.clone()
    holes[0, 3], holes[3, 1], holes[2, 0] = -1, 10 ** 6, -1
    for tab in (table, holes):
        for got in both(cache, tab):
            _compare(got, q, cache, tab, lengths, counts)
    clean = both(cache, table)[0]
    last = int(table[3, 299 // page])
    cache.k.view(torch.uint8)[last, :, 300 % page:] = 0x7f   # behind the sequence: not seen
    cache.v.view(torch.uint8)[last, :, :, 300 % page:] = 0xff
    for got in both(cache, table):
        _compare(got, q, cache, table, lengths, counts)
    assert all(torch.equal(x, y) for x, y in zip(both(cache, table)[0], clean))
    at = 300 - 20   # seen by the last 20 new tokens
    cache.v.view(torch.uint8)[int(table[3, at // page]), 1, d - 3, at % page] = 0x7f
    cache.v.view(torch.uint8)[int(table[0, 0]), 0, 5, 9] = 0xff   # by all
    cache.k.view(torch.uint8)[int(table[2, 0]), 1, 2, 7] = 0x7f
    cache.v_scale[int(table[0, 600 // page]), 1] = math.nan
    wide, few, parts, groups = both(cache, table)
    for got in (wide, parts, groups):
        for x, y in zip(got, few):
            assert torch.equal(x.isnan(), y.isnan())
    sees = torch.arange(300 - 33, 300) >= at
    assert torch.equal(wide[0][3, 3, :33, d - 3].isnan(), sees) and not bool(wide[0][3, :3].isnan().any())
    assert bool(wide[0][0, :3, :, 5].isnan().all()) and bool(wide[0][0, 3:].isnan().all())
    assert bool(wide[0][2, 3:, :7].isnan().all()) and not bool(wide[0][2, :3].isnan().any())


@pytest.mark.parametrize("batch,heads,d", [(700, 2, 64), (1100, 2, 64), (1100, 2, 128), (800, 20, 64), (800, 20, 128)])
def test_more_sequences_than_threads(gpu, batch, heads, d):
    lengths = [(i * 37) % 90 for i in range(batch)]
    cache, table = _cache(batch, 1, 16, d, 40, lengths)
    q = seeded_normal((batch, heads, 1, d), 5)
    _compare(_run(q, _gpu(cache), table, lengths), q, cache, table, lengths)


@pytest.mark.parametrize("tokens", [1, 6, 80])
def test_pages_the_cache_does_not_have(gpu, tokens):
    cache, table = _cache(2, 2, 16, 64, 20, (300, 200))
    table[0, 3], table[0, 18], table[1, 0], table[1, 1] = -1, 10 ** 6, -2 ** 31, 2 ** 31 - 1
    q = seeded_normal((2, 4, tokens, 64), 5)
    for lengths in ((300, 200), (320, 32), (2 ** 31 - 1, -7)):
        _compare(_run(q, _gpu(cache), table, lengths), q, cache, table, lengths)
    _compare(_run(q, _gpu(cache), table, (300, 200), (-4, 2 ** 31 - 1)), q, cache, table, (300, 200), (-4, 2 ** 31 - 1))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("tokens", [1, 5, 70])
def test_what_lies_behind_a_sequence_is_not_seen(gpu, tokens, d):
    """NaN codes and scales past the end, and in the keys and values of later tokens, for the rows before them."""
    length = 150
    cache, table = _cache(1, 1, 32, d, 6, (length,))
    q = seeded_normal((1, 3, tokens, d), 5)
    want = _run(q, _gpu(cache), table, (length,))
    last = int(table[0, 4])
    cache.k.view(torch.uint8)[last, :, length % 32:] = 0x7f
    cache.v.view(torch.uint8)[last, :, :, length % 32:] = 0xff
    for p in range(cache.k.shape[0]):
        if p not in table[0].tolist():
            cache.k_scale[p], cache.v_scale[p] = math.nan, math.inf
    got = _run(q, _gpu(cache), table, (length,))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    if tokens == 1:
        return
    at = length - 2   # one value, then one key of the token before the last
    for which in "vk":
        bad = api.KVCache(*(x.clone() for x in cache))
        if which == "v":
            bad.v.view(torch.uint8)[last, 0, 7, at % 32] = 0xff
        else:
            bad.k.view(torch.uint8)[last, 0, at % 32, 9] = 0x7f
        o, lse = (x.cpu() for x in _run(q, _gpu(bad), table, (length,)))
        sees = torch.arange(length - tokens, length) >= at
        assert torch.equal(o[:, :, ~sees], want[0].cpu()[:, :, ~sees])
        assert torch.equal(lse[:, :, ~sees], want[1].cpu()[:, :, ~sees])
        if which == "v":
            hit = torch.arange(d) == 7
            assert bool(o[:, :, sees][..., hit].isnan().all()) and torch.equal(lse, want[1].cpu())
            assert torch.equal(o[:, :, sees][..., ~hit], want[0].cpu()[:, :, sees][..., ~hit])
        else:
            assert bool(o[:, :, sees].isnan().all()) and bool(lse[:, :, sees].isnan().all())


def test_nan_of_a_key_or_value_that_all_rows_see(gpu):
    cache, table = _cache(1, 2, 16, 64, 12, (180,))
    cache.v.view(torch.uint8)[int(table[0, 2]), 0, 3, 5] = 0x7f
    cache.k.view(torch.uint8)[int(table[0, 2]), 1, 6, 5] = 0x7f
    q = seeded_normal((1, 2, 1, 64), 5)
    o, lse = (x.cpu() for x in _run(q, _gpu(cache), table, (180,)))
    assert torch.equal(o[0, 0, 0].isnan(), torch.arange(64) == 3) and bool(lse[0, 0].isfinite().all())
    assert bool(o[0, 1].isnan().all()) and bool(lse[0, 1].isnan().all())
    q[0, 0, 0, 0] = math.nan
    o, lse = (x.cpu() for x in _run(q, _gpu(cache), table, (180,)))
    assert bool(o[0, 0].isnan().all()) and bool(lse[0, 0].isnan().all())


def test_large_scores(gpu):
    """Scores of thousands, and scales far from 1: the softmax runs on its running maximum."""
    cache, table = _cache(2, 1, 16, 64, 20, (300, 77))
    cache.k_scale.mul_(2.0 ** 9)
    cache.v_scale.mul_(2.0 ** -60)
    q = seeded_normal((2, 2, 1, 64), 5)
    o, lse, weight = attention_cached_ref(q, cache, table, (300, 77))
    got = _run(q, _gpu(cache), table, (300, 77))
    # a score is off by at most (D + 4) * 2^-24 * sum |q k| / 8, and a probability by as much
    _, k_size, _ = attention_cached_ref(q.abs(), api.KVCache(cache.k.float().abs().to(cache.k.dtype), *cache[1:]), table, (300, 77))
    part = 2.0 ** -16.9 * k_size[..., None] + 2 ** -8
    assert bool(((got[0].cpu().double() - o).abs() <= 2 ** -8 * o.abs() + part * weight).all())
    assert bool(((got[1].cpu().double() - lse).abs() <= 2.0 ** -16.9 * k_size).all())


def test_shared_pages_and_strided_tensors(gpu):
    """Two sequences over one prefix; q, out and lse as views; a workspace that is given."""
    cache, table = _cache(2, 2, 32, 128, 6, (192, 192))
    table[1, :4] = table[0, :4]
    q = seeded_normal((2, 3, 10, 128), 5).cuda().permute(0, 2, 1, 3)[:, 2:6]     # [2, 4, 3, 128]
    wide = torch.full((2, 3, 8, 128), 5.0, dtype=torch.bfloat16, device="cuda").permute(0, 2, 1, 3)
    lse = torch.full((2, 4, 3, 2), 5.0, device="cuda")
    tables = torch.nn.functional.pad(table, (1, 3), value=-1).cuda()[:, 1:7]
    g = _gpu(cache)
    ws = torch.full((api.attention_cached_workspace(q, g, tables) + 8,), math.nan, device="cuda")
    got = api.attention_cached(q, g, tables, _ints((192, 150)).cuda(), out=wide[:, 1:5], lse=lse[..., 0], workspace=ws)
    _compare(got, q, cache, table, (192, 150))
    assert bool((wide[:, [0, 5, 6, 7]] == 5).all()) and bool((lse[..., 1] == 5).all()) and bool(ws[-8:].isnan().all())
    for _ in range(2):
        got = api.attention_cached(q, g, tables, _ints((192, 150)).cuda(), out=wide[:, 1:5], lse=lse[..., 0])
        _compare(got, q, cache, table, (192, 150))


def test_nothing_to_do(gpu):
    g = api.KVCache.empty(2, 2, 16, 64)
    q = seeded_normal((3, 4, 2, 64), 0).cuda()
    o, lse = api.attention_cached(q, g, torch.zeros(3, 0, dtype=torch.int32, device="cuda"), _ints((1, 2, 3)).cuda())
    assert bool((o == 0).all()) and bool((lse == -math.inf).all())
    for bad in (q[:0], q[:, :, :0]):
        o, lse = api.attention_cached(bad, g, torch.zeros(bad.shape[0], 2, dtype=torch.int32, device="cuda"),
                                      _ints([1] * bad.shape[0]).cuda())
        assert o.shape == bad.shape and lse.shape == bad.shape[:3]


def test_offsets_past_32_bits(gpu):
    page, d, h = 128, 128, 8
    pages = 2 ** 32 // (page * d * h) + 3
    big = api.KVCache.empty(pages, h, page, d)
    small, table = _cache(1, h, page, d, 2, (200,), spare=0)
    at = (pages - 1, pages - 2)
    for i, p in enumerate(at):
        for x, y in zip(big, small):
            x.view(torch.uint8 if x.dtype != torch.float32 else x.dtype)[p] = \
                y.view(torch.uint8 if x.dtype != torch.float32 else x.dtype)[i].cuda()
    far = torch.tensor([[at[int(table[0, 0])], at[int(table[0, 1])]]], dtype=torch.int32)
    for tokens in (1, 20):
        q = seeded_normal((1, 16, tokens, d), 1)
        got, want = _run(q, big, far, (200,)), _run(q, _gpu(small), table, (200,))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and bool((got[0] != 0).any())


def test_streams_and_graphs(gpu):
    """A decode loop's two calls, captured: every replay is the eager result, also with eager work between."""
    cache, table = _cache(3, 2, 16, 64, 60, (900, 20, 0))
    table = torch.arange(180, dtype=torch.int32).view(3, 60)
    g, t = _gpu(cache), table.cuda()
    lengths = _ints((901, 21, 1)).cuda()
    q, k, v = (seeded_normal((3, h, 1, 64), s).cuda() for s, h in enumerate((8, 2, 2)))
    start = [x.clone() for x in g]

    def step():
        api.kv_cache_write(g, k, v, t, lengths)
        return api.attention_cached(q, g, t, lengths)

    def feed(n):
        lengths.copy_(_ints((901 + n, 21 + n, 1 + n)))
        for i, x in enumerate((q, k, v)):
            x.copy_(seeded_normal(x.shape, 10 * n + i).cuda())

    eager = []
    for n in range(6):
        feed(n)
        eager.append([x.clone() for x in step()])
    for x, y in zip(g, start):
        x.copy_(y)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        held = step()
    for n in range(6):
        feed(n)
        if n % 2:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                got = step()
            torch.cuda.current_stream().wait_stream(side)
        else:
            graph.replay()
            got = held
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, eager[n]))
