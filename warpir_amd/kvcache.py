"""Keys and values in 8 bits: the paged cache, its write and read
(``csrc/kv_cache.hip``) and attention over it (``csrc/attn_cached.hip``)."""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Tuple

from warpir_amd.handwritten import DevicePlans, check_tensor, check_written, launch, need

PAGE_SIZES = (16, 32, 64, 128)
_write_plans = DevicePlans("kv_cache_write")
_read_plans = DevicePlans("kv_cache_read")


class KVCache(NamedTuple):
    """A paged cache of keys and values in e4m3 codes (``torch.float8_e4m3fn``)
    with one fp32 scale for each page and key/value head; a code stands for
    ``code * scale``.  Tokens lie next to one another in a V page, since
    attention's second product sums over them."""

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
    launch(rec, device, "kv_cache.hsaco", f"{kernel}_d{d}", (programs, 1, 1), (256, 1, 1), args,
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
    that is written may belong to one sequence only: two that write it at once
    leave a mixture of both there."""
    import torch

    fn, done = "kv_cache_write", None
    planned = isinstance(cache, KVCache)
    if planned:
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


__all__ = ["KVCache", "kv_cache_write", "kv_cache_read"]
