"""Keys and values in 8 bits: the paged cache, its write and read
(``csrc/kv_cache.hip``) and attention over it (``csrc/attn_cached.hip``)."""
from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple, Tuple

from warpir_amd.handwritten import DevicePlans, apart, check_tensor, check_written, launch, need, own

PAGE_SIZES = (16, 32, 64, 128)
_write_plans = DevicePlans("kv_cache_write")
_read_plans = DevicePlans("kv_cache_read")
_attention_plans = DevicePlans("attention_cached")


class KVCache(NamedTuple):
    """A paged cache of keys and values in e4m3 codes (``torch.float8_e4m3fn``)
    with one fp32 scale for each page and key/value head; a code stands for
    ``code * scale`` (scales are positive).  Tokens lie next to one another in a V
    page, since attention's second product sums over them."""

    k: object        # [pages, H_kv, page size, D]
    v: object        # [pages, H_kv, D, page size]
    k_scale: object  # [pages, H_kv]
    v_scale: object  # [pages, H_kv]

    @staticmethod
    def empty(pages: int, kv_heads: int, page_size: int, d: int, device="cuda") -> "KVCache":
        """A cache of zeros."""
        import torch

        need("KVCache.empty", pages > 0 and kv_heads > 0 and page_size in PAGE_SIZES and d in (64, 128),
             f"pages and kv_heads must be positive, page_size one of {PAGE_SIZES}, d 64 or 128")
        return KVCache(*(torch.zeros(pages, kv_heads, *page, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
                         for page in ((page_size, d), (d, page_size))),
                       *(torch.zeros(pages, kv_heads, dtype=torch.float32, device=device) for _ in "kv"))


class _Side(ctypes.Structure):
    _fields_ = [("codes", ctypes.c_void_p), ("scales", ctypes.c_void_p), ("x", ctypes.c_void_p),
                *((n, ctypes.c_longlong) for n in ("xb", "xh", "xt"))]


class _Args(ctypes.Structure):
    _fields_ = [("k", _Side), ("v", _Side), ("table", ctypes.c_void_p), ("lengths", ctypes.c_void_p),
                ("counts", ctypes.c_void_p), ("tb", ctypes.c_longlong),
                *((n, ctypes.c_int) for n in ("batch", "heads", "tokens", "page", "pages", "columns", "slots"))]


def _validate(fn, cache, page_table, lengths, counts):
    """(batch, kv_heads, page size, D, device) of a cache and the sequences in it."""
    import torch

    if not isinstance(cache, KVCache):
        raise TypeError(f"{fn}: cache must be a KVCache")
    codes, device = torch.float8_e4m3fn, getattr(cache.k, "device", None)
    check_tensor(fn, "cache.k", cache.k, codes, (None,) * 4, None)
    pages, heads, page, d = cache.k.shape
    need(fn, page in PAGE_SIZES, f"the page size must be one of {PAGE_SIZES}, got {page}")
    need(fn, d in (64, 128), f"the head size must be 64 or 128, got {d}")
    need(fn, pages > 0 and heads > 0, "the cache has no pages or heads")
    check_tensor(fn, "cache.v", cache.v, codes, (pages, heads, d, page), device)
    for name, s in (("cache.k_scale", cache.k_scale), ("cache.v_scale", cache.v_scale)):
        check_tensor(fn, name, s, torch.float32, (pages, heads), device, rows=False)
    for name, t in zip(KVCache._fields, cache):
        need(fn, t.is_contiguous(), f"cache.{name} must be contiguous")
    need(fn, pages < 1 << 31 and heads * page * d < 1 << 31, "a page or the number of pages does not fit in 31 bits")
    check_tensor(fn, "page_table", page_table, torch.int32, (None, None), device, rows=False)
    batch, columns = page_table.shape
    need(fn, columns == 0 or batch == 0 or page_table.stride(1) == 1 or columns == 1,
         "page_table's last dimension must be contiguous")
    need(fn, columns * page <= 1 << 30, "page_table holds more than 2^30 tokens a sequence")
    check_tensor(fn, "lengths", lengths, torch.int32, (batch,), device, rows=False)
    need(fn, batch <= 1 or lengths.stride(0) == 1, "lengths must be contiguous")
    if counts is not None:
        check_tensor(fn, "counts", counts, torch.int32, (batch,), device, rows=False)
        need(fn, batch <= 1 or counts.stride(0) == 1, "counts must be contiguous")
    return batch, heads, page, d, device


def _launch(fn, rec, kernel, cache, k, v, page_table, lengths, counts, slots, device):
    batch, heads, tokens, d = k.shape
    programs = batch * slots * heads * 2
    need(fn, programs < 1 << 24, "2^24 pages or more in one call")
    if not programs:
        return False
    args = _Args(*(_Side(None, None, None, *x.stride()[:3]) for x in (k, v)), None, None, None, page_table.stride(0),
                 batch, heads, tokens, cache.k.shape[2], cache.k.shape[0], page_table.shape[1], slots)
    lanes = cache.k.shape[2] // 4 * (d // 8)   # of a page: 4 tokens x 8 columns each
    kind = "_packed" if lanes <= 64 else "_p128" if lanes > 256 else ""
    if lanes <= 64:   # pages of a workgroup (csrc/kv_cache.hip)
        programs = -(-programs * lanes // 256)
    launch(rec, device, "kv_cache.hsaco", f"{kernel}_d{d}{kind}", (programs, 1, 1), (256, 1, 1), args,
           {"k.codes": cache.k, "k.scales": cache.k_scale, "k.x": k, "v.codes": cache.v, "v.scales": cache.v_scale,
            "v.x": v, "table": page_table, "lengths": lengths, "counts": counts})
    return True


def kv_cache_write(cache: KVCache, k, v, page_table, lengths, counts=None) -> KVCache:
    """Quantise new keys and values ``[B, H_kv, T, D]`` (bf16) into ``cache``, in
    place; returns ``cache``.

    Sequence ``b`` holds ``lengths[b]`` tokens with the new ones, its last
    ``counts[b]`` of them (default T) are tokens ``0 .. counts[b] - 1`` of ``k[b]``
    and ``v[b]``; what lies behind those is not read.  Position ``p`` lies in page
    ``page_table[b, p // page_size]`` (int32 ``[B, columns]``; ``lengths`` and ``counts``
    are int32).

    A page's scale is the smallest power of two that holds its values' largest
    magnitude in e4m3's 448.  Tokens that join a page which already holds some
    keep its scale if it is large enough; where it has to grow, the page's codes
    are rounded again for the new one.  An infinity becomes NaN, which e4m3 has.
    Nothing else in the cache changes.  Tokens before position 0, past the
    table, or in a page that the cache does not have (-1) are dropped.  A page
    that is written stands in one place of the table only: tokens that reach it
    by two (sequences, or columns of one) leave a mixture of both there."""
    import torch

    fn, done = "kv_cache_write", None
    if counts is lengths:
        counts = own(counts, lengths)
    if isinstance(cache, KVCache):
        need(fn, cache.k_scale is not cache.v_scale, "cache.k_scale and cache.v_scale are one tensor")
        done = _write_plans.run(0, k, v, *cache, page_table, lengths, counts)
        if done is not None and done is not False:
            return cache
    batch, heads, page, d, device = _validate(fn, cache, page_table, lengths, counts)
    check_tensor(fn, "k", k, torch.bfloat16, (batch, heads, None, d), device)
    check_tensor(fn, "v", v, torch.bfloat16, k.shape, device)
    tokens = k.shape[2]
    need(fn, tokens <= 1 << 30, "more than 2^30 tokens")
    rec = _write_plans.recording(done, k, v, *cache, page_table, lengths, counts)
    slots = min((tokens + page - 2) // page + 1, page_table.shape[1]) if tokens else 0
    ran = _launch(fn, rec, "wir_kv_write", cache, k, v, page_table, lengths, counts, slots, device)
    if rec and ran:
        _write_plans.add(0, rec, cache.k)
    return cache


def kv_cache_read(cache: KVCache, page_table, lengths, tokens: int, k=None, v=None) -> Tuple[object, object]:
    """The first ``tokens`` places of every sequence as dense bf16 ``(k, v)``,
    ``[B, H_kv, tokens, D]`` (allocated if omitted), as ``api.attention_forward`` takes
    them.  Places past a sequence's length, past the table, or in a page that
    the cache does not have become 0."""
    import torch

    fn, done = "kv_cache_read", None
    need(fn, k is None or k is not v, "k and v are one tensor")
    if k is not None and v is not None:
        apart(fn, ("k", "v"), 1, k, v)
    if isinstance(cache, KVCache) and type(tokens) is int:
        done = _read_plans.run(tokens, *cache, page_table, lengths, k, v)
        if done is not None and done is not False:
            return done
    batch, heads, page, d, device = _validate(fn, cache, page_table, lengths, None)
    if not isinstance(tokens, int) or isinstance(tokens, bool) or not 0 <= tokens <= 1 << 30:
        raise ValueError(f"{fn}: tokens must be an int from 0 to 2^30, got {tokens!r}")
    rec = _read_plans.recording(done, *cache, page_table, lengths, k, v)
    outs = []
    for name, x in (("k", k), ("v", v)):
        if x is None:
            x = rec.alloc(torch.empty(batch, heads, tokens, d, dtype=torch.bfloat16, device=device))
        check_tensor(fn, name, x, torch.bfloat16, (batch, heads, tokens, d), device)
        check_written(fn, name, x)
        outs.append(x)
    ran = _launch(fn, rec, "wir_kv_read", cache, *outs, page_table, lengths, None, -(-tokens // page), device)
    if rec and ran:
        _read_plans.add(tokens, rec, *outs)
    return outs[0], outs[1]


class _AttnArgs(ctypes.Structure):
    _fields_ = [*((n, ctypes.c_void_p) for n in ("q", "k", "v", "k_scale", "v_scale", "table", "lengths", "counts",
                                                 "out", "lse", "partial", "info")),
                *((n, ctypes.c_longlong) for n in ("qb", "qh", "qt", "ob", "oh", "ot", "lb", "lh", "lt", "tb")),
                *((n, ctypes.c_int) for n in ("batch", "heads", "group", "tokens", "page_shift", "pages", "columns",
                                              "blocks", "extra", "least"))]


TILE = 64        # positions of a tile (csrc/wir_pages.h)


# us of one tile of a workgroup that has a CU to itself, and of one CU's time where all are busy, by head size and rows
# of a block: the slopes of launches of 30 to 500 tiles
_TILE_US = {128: {16: (0.35, 0.35), 32: (0.55, 0.43), 128: (1.2, 1.1)},
            64: {16: (0.22, 0.125), 32: (0.29, 0.18), 128: (0.85, 0.62)}}
_DIVIDED_US = {128: (13, 0.5, 24, 1.23), 64: (13, 0.26, 24, 0.75)}   # divided: us, and us of a CU for a tile; 16, 128


@functools.lru_cache(maxsize=1024)
def _attention_form(rows: int, heads: int, columns: int, page: int, d: int):
    """(rows of a block, waves, extra, least) of the kernel for ``rows`` query
    rows a key/value head over a table of ``columns`` pages, ``heads`` of them in all
    sequences together.  The heads' tiles are divided over at most ``extra`` more
    programs than one for each (sequence, block, head), in parts of at least
    ``least`` tiles; extra 0: no division.  A division adds up the tiles in 32 bits
    (2^30 of them at most) and joins rows in a launch of its own: past either's
    bound the form's kernel runs undivided."""
    block, waves, extra, least = _fastest_form(rows, heads, columns, page, d)
    items = heads * -(-rows // block)
    if extra and (items * max(1, -(-columns * page // TILE)) >= 1 << 30 or
                  _join_grid(items, rows, block)[0] >= 1 << 24):
        return block, waves, 0, 0
    return block, waves, extra, least


def _join_grid(items: int, rows: int, block: int):
    """(workgroups of 256, whether a wave takes a row) of the launch that joins ``items`` blocks' partial results."""
    each = min(rows, block)
    if block == 128 and items * each > 2048:
        return items * -(-each // 4), True
    return items * each, False


def _attention_kernels(block: int, waves: int, extra: int, d: int, page: int, many: bool):
    """Names of the launches of a form: attention and, where heads are divided, the join."""
    kind = ("" if waves == 4 else f"_w{waves}") + ("_p64" if block == 128 and page >= TILE else "")
    names = [f"wir_attn_cached_d{d}_r{block}{kind}"]
    return names + [f"wir_attn_join_d{d}_r{block}" + ("_w4" if many else "")] if extra else names


def _fastest_form(rows: int, heads: int, columns: int, page: int, d: int):
    """The form of ``_attention_form`` by time.

    Up to 32 rows, one block: a division costs a second launch and the partial
    results' way, ~3 us; a head that is not divided is read by one CU at ~49
    GB/s, against ~5 TB/s of the chip, so it pays below ~105 heads and from ~150
    kB of keys and values in a head, or where one sequence may be far longer
    than the rest.  us, divided / not (8 heads of D = 128 a sequence): 1 x 1000
    keys 11.1 / 10.9, 1 x 4000 11.2 / 26.6, 4 x 2048 13.7 / 17.5, 16 x 2048 20.5 / 17.9,
    32 x 512 12.8 / 9.7; 16 x 16 heads of D = 64, up to 2050 keys 16.6 / 13.4.

    More rows: the form with the smallest estimate for keys that fill the
    table.  Blocks of 16 rows win while they leave CUs idle, blocks of 128 where
    the work is much.  us, 16 / 32 / 128 rows / 16 divided / 128 divided (D = 128,
    H32/8): 16 queries over 8000 keys 53.6 / 83 / 193 / 19.2 / 24.7, 40 over 2000 17.1 /
    26 / 60 / 19.7 / 25, 8 x 64 over 2000 54 / 41.8 / 54 / - / 50, 64 over 32000 193 / 296 /
    649 / 111 / 68, 2 x 1000 over 8192 665 / 430 / 278 / - / 293."""
    if rows > 32:
        tiles = -(-columns * page // TILE)
        n = {block: heads * -(-rows // block) for block in (16, 32, 128)}
        each = {block: x / 256 if x > 512 else -(-x // 256) for block, x in n.items()}   # programs of a CU
        # of later programs (beside their tiles; by launches of 512 to 16384 blocks of 16 / 32 / 128 rows with one tile
        # each: 3.7 / 6.9 / 8.5 us for 512 at D = 128, 1.7 / 4.1 / 4.2 at 64)
        starts = {block: (6 if d == 128 else 3) * max(x / 512 - 1, 0) for block, x in n.items()}
        us = {(block, 0): 6 + starts[block] + tiles * max(light, busy * each[block])
              for block, (light, busy) in _TILE_US[d].items()}
        few, few_tile, many, many_tile = _DIVIDED_US[d]
        # (past two programs a CU a division only adds to the starts, which these leave out, and to what each program
        # adds up; us, divided / not: 64 x 300 queries over 400 keys (32/8 heads, D = 128) 356 / 198, 500 x 64 over 100 (64/4)
        # 2577 / 423, 100 x 1000 over 1000 (128/16) 24700 / 5250; D = 64: 64 x 300 over 400 (64/4) 770 / 204)
        if n[16] <= 512:
            us[16, 1] = few + few_tile * max(n[16] * tiles / 256, 2)
        if n[128] <= 512:
            us[128, 1] = many + many_tile * max(n[128] * tiles / 256, 2)
        block, divided = min(us, key=us.get)
        if divided:
            return block, 4, 256 if block == 16 else max(512 - n[128], 256), 2
        # a CU's only block of 128 rows: its tiles divided over two groups of four waves (us, 1 x 1000 queries over 8192 keys
        # 180 / 156, 1909 over 1914, 16/16 heads, 52 / 44)
        return block, 8 if block == 128 and n[128] <= 256 else 4, 0, 0
    block, held = 16 if rows <= 16 else 32, columns * page * 2 * d   # bytes of a head at most
    if held <= 640 << 10 and held * (1 - heads / 105) <= 147 << 10:
        # eight waves a head while there is one such program for each CU, two where more heads than four fill the CUs
        # with are short (us, two / four waves, 32/8 heads of D = 128: 1024 sequences of up to 200 keys 67 / 92, 128 of up to
        # 1000 32.0 / 32.3, 100 of up to 300 13.1 / 15.3; with 8 tokens 512 of up to 1000 164 / 180, 128 of 1000 47.5 / 55;
        # but 512 of up to 2500 249 / 242, and with 8 tokens 80 of up to 1000 41 / 37)
        short = columns * page <= 16 * TILE
        if heads >= 768 and short:
            return block, 2, 0, 0
        return block, 8 if heads <= 256 and not short and (block, d) != (32, 128) else 4, 0, 0
    # more heads than 512 fill the chip by themselves, and every program of a division adds up all sequences' tiles: the
    # kernel runs undivided.  us, divided / not (32/8 heads, D = 128, lengths from 1 to the named, in a table of 32768):
    # 1024 sequences of 200 keys 536 / 145, of 4000 1047 / 739, 96 of 200 28.8 / 15.2, of 8192 166 / 160; with 8 tokens 512 of
    # 1000 278 / 177; 16/16 heads, D = 64: 512 of 1000 230 / 117.  (One of 32000 among 511 of 200: 198 / 238.)
    if heads > 512:
        return block, 4 if (block, d) == (32, 128) else 8, 0, 0
    # two programs of four waves a CU (32 sequences of up to 16000 keys, 256 heads: 384 more 96.6, 128 or 1024 over
    # 99); with more heads, one of eight and as many more (64 sequences of up to 8192, 512 heads: 512 more of eight
    # waves 119.6, 1536 of four 122)
    if heads <= 384 or (block, d) == (32, 128):
        return block, 4, max(512 - heads, 384), 2
    return block, 8, 512, 2


def attention_cached(q, cache: KVCache, page_table, lengths, counts=None, out=None, lse=None,
                     workspace=None) -> Tuple[object, object]:
    """Attention of new queries ``[B, H, T, D]`` (bf16, H a multiple of the
    cache's heads) over a paged cache; returns ``(O, LSE)``, bf16 ``[B, H, T, D]`` and
    fp32 ``[B, H, T]`` (natural log), as ``api.attention_forward``.

    The sequences are as in ``kv_cache_write``, which has put the new tokens'
    keys and values there: query ``t < counts[b]`` (default T) has position
    ``lengths[b] - counts[b] + t`` and sees the positions up to its own.  Keys in
    pages that the cache does not have (-1) are seen by no row.  A row that
    sees no key (also ``t >= counts[b]``, or a position below 0) gives O = 0 and
    LSE = -inf.

    The kernel is chosen by the shapes and the table's width, so the table
    should have the columns that the sequences may fill.  Where few heads leave
    CUs idle, the keys are divided over the chip by the lengths as they are on
    the GPU; partial results go through ``workspace`` (fp32, as many
    elements as ``attention_cached_workspace`` says, allocated if omitted), which
    one call at a time may use: two streams, or two graphs that run at once,
    need one each.  ``out`` may be ``q`` itself.

    Refused are 2^24 query rows (T * H / H_kv) or more a key/value head of a
    sequence, and launches of 2^32 threads or more."""
    import torch

    fn, done = "attention_cached", None
    if out is not None:   # (its own rows of q a workgroup reads before it writes them)
        apart(fn, ("out", "lse", "out", "q"), 1, out, lse, out, q)
    if counts is lengths:
        counts = own(counts, lengths)
    if isinstance(cache, KVCache) and workspace is None:
        done = _attention_plans.run(0, q, *cache, page_table, lengths, counts, out, lse)
        if done is not None and done is not False:
            return done
    batch, heads, page, d, device = _validate(fn, cache, page_table, lengths, counts)
    check_tensor(fn, "q", q, torch.bfloat16, (batch, None, None, d), device)
    h, tokens = q.shape[1:3]
    need(fn, h > 0 and h % heads == 0, f"{h} query heads are not a multiple of {heads} key/value heads")
    group = h // heads
    need(fn, tokens * group < 1 << 24, "2^24 query rows or more a key/value head of a sequence")
    rec = _attention_plans.recording(done, q, *cache, page_table, lengths, counts, out, lse)
    if out is None:
        out = rec.alloc(torch.empty(q.shape, dtype=q.dtype, device=device))
    if lse is None:
        lse = rec.alloc(torch.empty(q.shape[:3], dtype=torch.float32, device=device))
    check_tensor(fn, "out", out, torch.bfloat16, q.shape, device)
    check_tensor(fn, "lse", lse, torch.float32, q.shape[:3], device, rows=False)
    for name, x in (("out", out), ("lse", lse)):
        check_written(fn, name, x)
    if batch * tokens == 0:
        return out, lse
    if page_table.shape[1] == 0:
        return out.zero_(), lse.fill_(float("-inf"))
    rows = tokens * group
    block, waves, extra, least = _attention_form(rows, batch * heads, page_table.shape[1], page, d)
    blocks = -(-rows // block)
    items = batch * blocks * heads
    need(fn, (items + extra) * waves < 1 << 26, "2^32 threads or more in one call")
    # (no bound of the kernels: were the table full, the launch would take the best part of an hour)
    need(fn, blocks * -(-page_table.shape[1] * page // TILE) < 1 << 30, "2^30 tiles of keys or more a key/value head")
    args = _AttnArgs(*[None] * 12, *q.stride()[:3], *out.stride()[:3], *lse.stride(), page_table.stride(0), batch, heads,
                     group, tokens, page.bit_length() - 1, cache.k.shape[0], page_table.shape[1], blocks, extra, least)
    floats = _workspace_floats(extra, block, d, items)
    if floats:
        if workspace is None:
            workspace = rec.alloc(torch.empty(floats, dtype=torch.float32, device=device))
        check_tensor(fn, "workspace", workspace, torch.float32, (None,), device)
        need(fn, workspace.numel() >= floats, f"workspace needs {floats} elements")
    else:
        workspace = None
    tensors = {"q": q, "k": cache.k, "v": cache.v, "k_scale": cache.k_scale, "v_scale": cache.v_scale,
               "table": page_table, "lengths": lengths, "counts": counts, "out": out, "lse": lse,
               "partial": workspace, "info": workspace}
    past = {"info": 4 * (floats - 4 * items)}
    grid, many = _join_grid(items, rows, block)
    names = _attention_kernels(block, waves, extra, d, page, many)
    launch(rec, device, "attn_cached.hsaco", names[0], (items + extra, 1, 1), (64 * waves, 1, 1), args, tensors, past)
    if extra:
        launch(rec, device, "attn_cached.hsaco", names[1], (grid, 1, 1), (256, 1, 1), args, tensors, past)
    if rec:
        _attention_plans.add(0, rec, out, lse)
    return out, lse


def _workspace_floats(extra: int, block: int, d: int, items: int) -> int:
    """Slots of partial results, each a block's unnormalised rows, maxima and
    sums, and four words of every (sequence, block, head)."""
    return (3 * extra + 2) * block * (d + 2) + 4 * items if extra else 0


def attention_cached_workspace(q, cache: KVCache, page_table) -> int:
    """Elements that ``attention_cached`` needs of a ``workspace`` for these tensors."""
    _, heads, page, d = cache.k.shape
    rows = q.shape[2] * (q.shape[1] // heads)

    block, _, extra, _ = _attention_form(rows, q.shape[0] * heads, page_table.shape[1], page, d)
    return _workspace_floats(extra, block, d, q.shape[0] * -(-rows // block) * heads)


__all__ = ["KVCache", "kv_cache_write", "kv_cache_read", "attention_cached", "attention_cached_workspace"]
