"""TEST INFRASTRUCTURE -- 64-bit oracles of the head norms with rotation, the
paged 8-bit cache and attention over it, from their definitions, on the CPU,
one row, page or head at a time; never used by the product."""
from __future__ import annotations

import math

import torch

E4M3 = torch.float8_e4m3fn


# ---------------------------------------------------------------------------
# norm and rotation
# ---------------------------------------------------------------------------
def angles_ref(positions, d, base=10000.0):
    """[..., d / 2] angles of the positions."""
    return positions.double()[..., None] * base ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)


def _pairs(x, interleaved):
    return (x[..., 0::2], x[..., 1::2]) if interleaved else x.chunk(2, -1)


def _unpair(a, b, interleaved):
    return torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)


def norm_rope_ref(x, w, angle, eps=1e-6, interleaved=False):
    """(out, bound): [B, H, S, D] with angle [B or 1, S, D / 2]; ``bound`` is
    |a| + |b| of the normed pair behind each output."""
    x, w = x.double(), w.double()
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w
    a, b = _pairs(y, interleaved)
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    size = a.abs() + b.abs()
    return _unpair(a * c - b * s, b * c + a * s, interleaved), _unpair(size, size, interleaved)


def norm_rope_bwd_ref(g, x, w, angle, eps=1e-6, interleaved=False):
    """(dx, dw, bound of dx, bound of dw): the bounds are the same sums over
    absolute values."""
    g, x, w = g.double(), x.double(), w.double()
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    a, b = _pairs(g, interleaved)
    gy = _unpair(a * c + b * s, b * c - a * s, interleaved)
    size = _unpair(a.abs() + b.abs(), a.abs() + b.abs(), interleaved)
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    xr = x * r
    dx = r * (gy * w - xr * (gy * w * xr).mean(-1, keepdim=True))
    bound = r * (size * w.abs() + xr.abs() * (size * w.abs() * xr.abs()).mean(-1, keepdim=True))
    return dx, (gy * xr).sum((0, 1, 2)), bound, (size * xr.abs()).sum((0, 1, 2))


# ---------------------------------------------------------------------------
# the cache
# ---------------------------------------------------------------------------
def e4m3_ref(x):
    """float64 values rounded to the nearest e4m3 value, ties to even, as codes; infinities are NaN."""
    x = x.double()
    m, e = torch.frexp(x.abs())                       # |x| = m 2^e, 0.5 <= m < 1
    step = torch.exp2(torch.clamp(e - 1, min=-6).double() - 3)
    y = torch.where(x.isfinite(), torch.round(x / step) * step, torch.full_like(x, math.nan))
    assert bool((y.isnan() | (y.abs() <= 448)).all())
    return y.float().to(E4M3)


def scale_ref(amax: float) -> float:
    e = -126
    while 448.0 * 2.0 ** e < amax:
        e += 1
    return 2.0 ** e


def cache_write_ref(cache, k, v, table, lengths, counts=None):
    """Writes into ``cache`` (CPU tensors k, v, k_scale, v_scale; fields as the product's)."""
    kc, vc, ks, vs = cache
    pages, heads, page, _ = kc.shape
    for b in range(k.shape[0]):
        n = k.shape[2] if counts is None else min(max(int(counts[b]), 0), k.shape[2])
        length = max(int(lengths[b]), 0)
        start = length - n
        places = {}
        for t in range(n):
            if 0 <= start + t < table.shape[1] * page:
                places.setdefault((start + t) // page, []).append(t)
        for place, tokens in places.items():
            page_id = int(table[b, place])
            if not 0 <= page_id < pages:
                continue
            first = start + tokens[0] - place * page    # slot of the first new token
            for codes, scales, x in ((kc, ks, k), (vc.transpose(2, 3), vs, v)):
                for h in range(heads):
                    vals = x[b, h, tokens].double()
                    fine = vals[vals.isfinite()].abs()
                    scale, was = scale_ref(float(fine.max()) if fine.numel() else 0.0), float(scales[page_id, h])
                    held = codes[page_id, h]
                    if first > 0:
                        scale = was if was >= scale else scale
                        if scale != was:
                            held.view(torch.uint8)[:first] = e4m3_ref(held[:first].double() * (was / scale)).view(torch.uint8)
                    held.view(torch.uint8)[first:first + len(tokens)] = e4m3_ref(vals / scale).view(torch.uint8)
                    scales[page_id, h] = scale


def cache_read_ref(cache, table, lengths, tokens):
    """(k, v) in float64 [B, heads, tokens, D] and which places hold a token [B, tokens]."""
    kc, vc, ks, vs = cache
    pages, heads, page, d = kc.shape
    n = len(lengths)
    there = torch.zeros(n, tokens, dtype=torch.bool)
    outs = [torch.zeros(n, heads, tokens, d, dtype=torch.float64) for _ in "kv"]
    for b in range(n):
        for p in range(min(int(lengths[b]), tokens, table.shape[1] * page)):
            page_id = int(table[b, p // page])
            if 0 <= page_id < pages:
                there[b, p] = True
                outs[0][b, :, p] = kc[page_id, :, p % page].double() * ks[page_id].double()[:, None]
                outs[1][b, :, p] = vc[page_id, :, :, p % page].double() * vs[page_id].double()[:, None]
    return outs[0], outs[1], there


def attention_cached_ref(q, cache, table, lengths, counts=None):
    """(O, LSE, weight): float64; ``weight`` is sum_j p_j |v_j| of every output."""
    b, h, t, d = q.shape
    capacity = table.shape[1] * cache[0].shape[2]
    k, v, there = cache_read_ref(cache, table, lengths, min(capacity, max([int(x) for x in lengths] + [0])))
    o, weight = (torch.zeros(b, h, t, d, dtype=torch.float64) for _ in range(2))
    lse = torch.full((b, h, t), -math.inf, dtype=torch.float64)
    group = h // cache[0].shape[1]
    for i in range(b):
        n = t if counts is None else min(max(int(counts[i]), 0), t)
        for j in range(n):
            pos = max(int(lengths[i]), 0) - n + j
            seen = there[i] & (torch.arange(there.shape[1]) <= pos)
            if not bool(seen.any()):
                continue
            for head in range(h):
                x = k[i, head // group, seen] @ q[i, head, j].double() / math.sqrt(d)
                p = torch.softmax(x, 0)
                lse[i, head, j] = torch.logsumexp(x, 0)
                o[i, head, j] = p @ v[i, head // group, seen]
                weight[i, head, j] = p @ v[i, head // group, seen].abs()
    return o, lse, weight
