"""The paged 8-bit cache's write and read against the 64-bit oracle: every
code, scale and value is equal, and nothing else changes."""
import pytest
import torch

from oracle.layer_ref import cache_read_ref, cache_write_ref
from oracle.torch_ref import seeded_normal
from tests.conftest import announce
from warpir_amd import api

pytestmark = pytest.mark.gpu


def _same(a, b):
    """Equal values, NaN at the same places (its sign is no value)."""
    a, b = a.cpu().float(), b.cpu().float()
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())


def _cache(pages, heads, page, d, seed=0):
    """A cache whose every byte says something (no NaN codes)."""
    gen = torch.Generator().manual_seed(seed)
    codes = [torch.randint(0, 256, s, generator=gen, dtype=torch.uint8) for s in
             ((pages, heads, page, d), (pages, heads, d, page))]
    codes = [torch.where(c & 127 == 127, c ^ 1, c).view(torch.float8_e4m3fn) for c in codes]
    scales = [2.0 ** torch.randint(-12, 3, (pages, heads), generator=gen).float() for _ in "kv"]
    return api.KVCache(*(x.cuda() for x in (*codes, *scales)))


def _table(b, columns, pages, seed=0):
    ids = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))[:b * columns]
    return ids.view(b, columns).int()


def _write_and_compare(cache, k, v, table, lengths, counts=None):
    ref = [x.cpu().clone() for x in cache]
    cache_write_ref(ref, k.cpu(), v.cpu(), table, lengths, counts)
    got = api.kv_cache_write(cache, k, v, table.cuda(), lengths.cuda(), counts=None if counts is None else counts.cuda())
    assert got is cache
    for name, x, y in zip(cache._fields, cache, ref):
        assert _same(x, y), name


def _ints(*x):
    return torch.tensor(x, dtype=torch.int32)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_writes_over_sequences(gpu, page, d):
    """A prompt, single tokens and chunks into the same pages, sequences of unequal length."""
    announce(f"kv write page {page} D{d}")
    b, h, columns = 3, 2, 5
    cache, table = _cache(b * columns + 2, h, page, d), _table(b, columns, b * columns + 2)
    lengths = torch.zeros(b, dtype=torch.int32)
    for step, (tokens, counts) in enumerate([(page + 7, (page + 7, 3, 0)), (1, None), (1, (1, 0, 1)), (page - 1, None),
                                             (5, (2, 5, 4)), (1, None), (2 * page, (0, 2 * page, 1))]):
        k = seeded_normal((b, h, tokens, d), step, 2.0 ** (step - 3)).cuda()   # scales that grow
        v = seeded_normal((b, tokens, 3 * h, d), 50 + step, 2.0 ** (2 - step)).cuda().permute(0, 2, 1, 3)[:, 2 * h:]
        n = torch.tensor(counts if counts else [tokens] * b, dtype=torch.int32)
        lengths = lengths + n
        for _ in range(2):   # the call and its plan (a write twice is a write once)
            _write_and_compare(cache, k, v, table, lengths, n if counts else None)


def test_values_at_the_borders(gpu):
    """Ties, subnormals, 448 times a power of two, zeros, infinities and NaN; and a page that grows over them."""
    page, d = 16, 64
    cache, table = _cache(4, 1, page, d), _table(1, 3, 4)
    base = torch.tensor([448.0, 449.0, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10, 17.0, 19.0, 0.0, -0.0, -448.0, 1.0625,
                         1.1875, 2.0 ** -6, 2.0 ** -6 - 2.0 ** -10, 464.0, -27.0])
    k = base.repeat(1, 1, 5, d // 16).view(1, 1, 5, d).bfloat16().cuda()
    for scale in (1.0, 2.0 ** -100, 2.0 ** 100, 2.0 ** -133):
        x = (k.float() * scale).bfloat16()
        _write_and_compare(cache, x, x * 0.5, table, _ints(5))
        _write_and_compare(cache, x[:, :, :1] * 3, x[:, :, 1:2] * 64, table, _ints(6))   # grows
        _write_and_compare(cache, x[:, :, :1] * 0, x[:, :, 1:2] * 0.001, table, _ints(7))   # keeps
    k[0, 0, 1, 3], k[0, 0, 2, 7], k[0, 0, 4, 0] = float("inf"), float("nan"), float("-inf")
    _write_and_compare(cache, k, k.clone(), table, _ints(5))
    _write_and_compare(cache, torch.full_like(k, float("nan")), torch.zeros_like(k), table, _ints(13))
    big = torch.full_like(k[:, :, :3], torch.finfo(torch.bfloat16).max)
    _write_and_compare(cache, big, -big, table, _ints(19))


def test_a_page_without_a_scale_yet(gpu):
    """Old scales of 0 and NaN, and one that is no power of two."""
    for old in (0.0, float("nan"), 0.3, 1e-30):
        cache, table = _cache(2, 2, 32, 64), _table(1, 1, 2)
        cache.k_scale.fill_(old), cache.v_scale.fill_(old)
        x = seeded_normal((1, 2, 3, 64), 1).cuda()
        ref = [t.cpu().clone() for t in cache]
        cache_write_ref(ref, x.cpu(), x.cpu(), table, _ints(9))
        api.kv_cache_write(cache, x, x, table.cuda(), _ints(9).cuda())
        assert _same(cache.k_scale, ref[2]) and _same(cache.v_scale, ref[3])
        # x * (1 / 0.3) against x / 0.3: two fp32 roundings, which flip a code only next to a tie
        assert (cache.k.cpu().float() - ref[0].float()).nan_to_num().abs().gt(0).float().mean() <= 1e-3


@pytest.mark.parametrize("d", [64, 128])
def test_what_has_no_place_is_dropped(gpu, d):
    """Pages of the table that the cache does not have, tokens past the table and before position 0."""
    cache, table = _cache(6, 2, 16, d), _table(3, 2, 6)
    table[0, 1], table[1, 0] = -1, 6
    table[2, 0] = 2 ** 31 - 1
    x = seeded_normal((3, 2, 40, d), 3).cuda()
    for lengths in (_ints(32, 32, 32), _ints(40, 33, 50), _ints(7, 20, 39), _ints(0, -5, 2 ** 31 - 1)):
        _write_and_compare(cache, x, x, table, lengths)
    _write_and_compare(cache, x, x, table, _ints(20, 20, 20), _ints(-3, 2 ** 31 - 1, 50))


def test_tables_of_any_width(gpu):
    cache = _cache(8, 1, 16, 64)
    wide = _table(2, 4, 8)
    x = seeded_normal((2, 1, 9, 64), 3).cuda()
    ref = [t.cpu().clone() for t in cache]
    cache_write_ref(ref, x.cpu(), x.cpu(), wide[:, :3], _ints(20, 9))
    api.kv_cache_write(cache, x, x, wide.cuda()[:, :3], _ints(20, 9).cuda())
    assert all(_same(a, b) for a, b in zip(cache, ref))
    before = [t.clone() for t in cache]
    api.kv_cache_write(cache, x, x, wide.cuda()[:, :0], _ints(20, 9).cuda())
    api.kv_cache_write(cache, x[:, :, :0], x[:, :, :0], wide.cuda(), _ints(20, 9).cuda())
    api.kv_cache_write(cache, x[:0], x[:0], wide.cuda()[:0], _ints(20, 9).cuda()[:0])
    assert all(_same(a, b) for a, b in zip(cache, before))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page,tokens", [(16, 1), (16, 70), (32, 33), (64, 200), (128, 130), (128, 3)])
def test_read(gpu, page, tokens, d):
    announce(f"kv read page {page} tokens {tokens} D{d}")
    columns = -(-tokens // page)
    cache, table = _cache(3 * columns + 1, 3, page, d), _table(3, columns, 3 * columns + 1)
    table[1, columns - 1] = -1
    for lengths in (_ints(tokens, tokens, tokens), _ints(0, 1, max(1, tokens - 3)), _ints(-1, 2 ** 31 - 1, tokens + 9)):
        k, v, _ = cache_read_ref([x.cpu() for x in cache], table, lengths, tokens)
        for _ in range(2):
            got = api.kv_cache_read(cache, table.cuda(), lengths.cuda(), tokens)
            assert torch.equal(got[0].cpu().double(), k) and torch.equal(got[1].cpu().double(), v)
    out = torch.full((3, tokens + 2, 6, d), 9.0, dtype=torch.bfloat16, device="cuda").permute(0, 2, 1, 3)
    got = api.kv_cache_read(cache, table.cuda(), lengths.cuda(), tokens, k=out[:, :3, :tokens], v=out[:, 3:, 1:tokens + 1])
    assert torch.equal(got[0].cpu().double(), k) and torch.equal(got[1].cpu().double(), v)
    assert bool((out[:, :3, tokens:] == 9).all()) and bool((out[:, 3:, [0, tokens + 1]] == 9).all())


def test_read_of_no_table_and_nan_codes(gpu):
    cache, table = _cache(2, 1, 16, 64), _table(1, 2, 2)
    k, v = api.kv_cache_read(cache, table.cuda()[:, :0], _ints(5).cuda(), 7)
    assert bool((k == 0).all()) and bool((v == 0).all())
    cache.k.view(torch.uint8).fill_(127)
    cache.v.view(torch.uint8)[:, :, :, 3] = 255
    k, v = api.kv_cache_read(cache, table.cuda(), _ints(5).cuda(), 7)
    assert bool(k[:, :, :5].isnan().all()) and bool((k[:, :, 5:] == 0).all())
    assert bool(v[:, :, 3].isnan().all()) and bool(v[:, :, [0, 1, 2, 4, 5, 6]].isfinite().all())


def test_offsets_past_32_bits(gpu):
    """Pages past 2^32 bytes of codes."""
    page, d, h = 128, 128, 8
    pages = 2 ** 32 // (page * d * h) + 3
    cache = api.KVCache.empty(pages, h, page, d)
    table = _ints([pages - 1, 0], [pages - 2, 1]).view(2, 2)
    x, y = seeded_normal((2, h, 130, d), 1).cuda(), seeded_normal((2, h, 130, d), 2).cuda()
    api.kv_cache_write(cache, x, y, table.cuda(), _ints(130, 130).cuda())
    small = api.KVCache(*(t[[pages - 1, 0, pages - 2, 1]].contiguous() if t.dtype == torch.float32 else
                          t.view(torch.uint8)[[pages - 1, 0, pages - 2, 1]].contiguous().view(t.dtype) for t in cache))
    ref = [t.cpu() for t in api.KVCache.empty(4, h, page, d, device="cpu")]
    near = _ints([0, 1], [2, 3]).view(2, 2)
    cache_write_ref(ref, x.cpu(), y.cpu(), near, _ints(130, 130))
    assert all(_same(a, b) for a, b in zip(small, ref))
    got = api.kv_cache_read(cache, table.cuda(), _ints(130, 130).cuda(), 130)
    want = api.kv_cache_read(small, near.cuda(), _ints(130, 130).cuda(), 130)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and bool((got[0] != 0).any())


def test_streams_and_graphs(gpu):
    cache, table = _cache(6, 2, 16, 64), _table(2, 3, 6).cuda()
    start = [x.clone() for x in cache]
    k, v = (seeded_normal((2, 2, 1, 64), s).cuda() for s in (1, 2))
    lengths = _ints(1, 1).cuda()

    def restore():
        for x, y in zip(cache, start):
            x.copy_(y)

    def step():
        api.kv_cache_write(cache, k, v, table, lengths)
        return api.kv_cache_read(cache, table, lengths, 40)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    restore()
    eager = []
    for n in range(1, 36):
        lengths.fill_(n)
        k.copy_(seeded_normal(k.shape, n).cuda())
        eager.append([x.clone() for x in step()])
    restore()
    side = torch.cuda.Stream()
    for n in range(1, 36):
        lengths.fill_(n)
        k.copy_(seeded_normal(k.shape, n).cuda())
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph.replay() if n % 2 else [h.copy_(x) for h, x in zip(held, step())]
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(x, y) for x, y in zip(held, eager[n - 1]))
