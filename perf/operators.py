"""The operators of a transformer layer around its projections and its dense
attention, each as a call with inputs, work and exact values: the plain form
in elementary torch operations, or (``own``) the framework's kernels.

A case is a plain dict.  ``op`` is the call:

* ``rope``: the norm of every query and key head and the rotation by its
  position, on views of one fused projection or on dense heads; with
  ``train`` the backward pass too -> (q, k[, dq, dk, dq_weight, dk_weight]).
* ``write``: new keys and values into a paged cache of e4m3 codes with one
  power-of-two scale per page and head -> the cache (codes and scales of K
  and V).
* ``read``: a cache's keys and values as dense bf16 -> (k, v).
* ``attend``: attention of a few or many new queries over such a cache
  -> (O, LSE).

K pages are ``[page, head, token, dim]``, V pages ``[page, head, dim, token]``.
"""
import math
import random

import torch

own = False

EPS = 1e-6
BASE = 10000.0
E4M3_MAX = 448.0


def _rope(batch, seq, heads, kv_heads, dim, **more):
    return {"op": "rope", "batch": batch, "seq": seq, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "train": False, "interleaved": False, "packed": True, "far": 0, **more}


def _write(batch, tokens, context, kv_heads, dim, page, **more):
    return {"op": "write", "batch": batch, "tokens": tokens, "context": context, "kv_heads": kv_heads, "dim": dim,
            "page": page, "ragged": False, **more}


def _read(batch, length, kv_heads, dim, page, **more):
    return {"op": "read", "batch": batch, "length": length, "kv_heads": kv_heads, "dim": dim, "page": page,
            "ragged": False, **more}


def _attend(batch, tokens, length, heads, kv_heads, dim, page, **more):
    return {"op": "attend", "batch": batch, "tokens": tokens, "length": length, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "ragged": False, **more}


def listed():
    return [
        # one decode step of a small batch at far positions: the call itself is most of the time
        _rope(8, 1, 32, 8, 128, far=100000, name="rope_decode"),
        # the prefill of a few prompts of odd length, pairs side by side
        _rope(3, 1337, 24, 8, 64, interleaved=True, name="rope_prefill_odd"),
        # a training layer: forward and backward
        _rope(8, 4096, 16, 16, 128, train=True, name="rope_train"),
        # every sequence of a serving batch appends one token
        _write(64, 1, 2000, 8, 128, 64, ragged=True, name="write_decode"),
        # prompts of unequal length enter the cache
        _write(8, 4096, 0, 8, 128, 64, ragged=True, name="write_prefill"),
        # one short sequence back as dense keys and values
        _read(1, 500, 8, 64, 16, name="read_small"),
        # a batch of contexts back as dense keys and values, for a dense prefill on top of them
        _read(16, 8192, 8, 128, 64, ragged=True, name="read_batch"),
        # the next token of one short chat
        _attend(1, 1, 1000, 32, 8, 128, 64, name="attend_decode_small"),
        # the next token of every sequence of a serving batch
        _attend(64, 1, 8192, 32, 8, 128, 64, ragged=True, name="attend_decode_batch"),
        # the next token after one very long context
        _attend(1, 1, 131072, 32, 8, 128, 64, name="attend_decode_long"),
        # a few drafted tokens at once, one key/value head per query head, small pages
        _attend(16, 4, 2050, 16, 16, 64, 16, ragged=True, name="attend_draft_d64"),
        # a chunk of two long prompts over what the cache holds of them
        _attend(2, 1000, 8192, 32, 8, 128, 64, name="attend_chunk"),
    ]


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("rope", "write", "read", "attend", "attend"))
    most = max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        kv_heads = rng.choice((1, 2, 4, 8, 12, 16))
        heads = kv_heads * rng.choice((1, 2, 3, 4, 8))
        dim, page, ragged = rng.choice((64, 128, 128)), rng.choice((16, 32, 64, 128)), rng.random() < 0.6
        if op == "rope":
            seq = rng.choice((1, _log(rng, 2, 8192)))
            c = _rope(_log(rng, 1, 256), seq, heads, kv_heads, dim, train=rng.random() < 0.5,
                      interleaved=rng.random() < 0.3, packed=rng.random() < 0.7, far=rng.choice((0, 0, 1000000)))
        elif op == "write":
            tokens = rng.choice((1, 1, _log(rng, 2, 8192)))
            c = _write(_log(rng, 1, 256), tokens, rng.choice((0, _log(rng, 1, 8192))), kv_heads, dim, page,
                       ragged=ragged)
        elif op == "read":
            c = _read(_log(rng, 1, 64), _log(rng, 1, 32768), kv_heads, dim, page, ragged=ragged)
        else:
            tokens = rng.choice((1, 1, rng.randint(2, 8), _log(rng, 9, 2048)))
            c = _attend(_log(rng, 1, 256), tokens, tokens + _log(rng, 1, 131072), heads, kv_heads, dim, page,
                        ragged=ragged)
        # (the plain form's scores and keys in 32 bits have to fit beside the inputs)
        size = c["batch"] * c.get("length", 1) * (heads * c.get("tokens", 1) + 8 * kv_heads * dim) if op == "attend" else 0
        if _cost(c) <= most and size <= 6e9 and c["batch"] * c.get("tokens", 1) <= 1 << 17:
            return c


def _lengths(case):
    """(length of every sequence with its new tokens, its new tokens): the batch of the case, whatever the seed."""
    n, t = case["batch"], case.get("tokens", 0)
    longest = case["context"] + t if case["op"] == "write" else case["length"]
    if not case["ragged"]:
        return [longest] * n, [t] * n
    rng = random.Random("%d %d %d" % (n, t, longest))
    lengths = [rng.randint(min(longest, max(1, t)), longest) for _ in range(n)]
    lengths[n // 2] = longest
    new = [t if t == 1 else min(x, rng.randint(1, max(1, t))) for x in lengths]
    if case["op"] == "write" and not case["context"]:
        new = lengths = [rng.randint(1, t) for _ in range(n)]
        new[n // 2] = t
    if n > 4:   # a slot of the batch that no sequence holds
        lengths[n // 4] = new[n // 4] = 0
    return lengths, new


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.bfloat16)


def _table(positions, dim):
    freq = BASE ** (-torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / dim)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _scale(amax):
    """The smallest 2^e with amax <= 448 * 2^e (2^-126 at least, also where amax is 0)."""
    mantissa, exponent = torch.frexp(amax.float() / 2)   # amax = 2 * mantissa * 2^exponent, 0.5 <= mantissa < 1
    e = exponent - 8 + (mantissa > 0.875).int()
    return (torch.where(amax > 0, e, -126).clamp(min=-126).int() + 127 << 23).view(torch.float32)


def _cache(gen, case, lengths):
    """A paged cache that holds sequences of these lengths, in pages of any order."""
    page, h, d = case["page"], case["kv_heads"], case["dim"]
    most = max(1, -(-max(lengths) // page))
    width = -(-most // 8) * 8
    used = [-(-x // page) for x in lengths]
    pages = max(1, sum(used)) + 3
    ids = torch.randperm(pages, generator=torch.Generator().manual_seed(int(gen.initial_seed())))[:max(1, sum(used))]
    held = torch.arange(width) < torch.tensor(used)[:, None]
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    table[held] = ids[:int(held.sum())].int()
    k = _normal(gen, pages, h, page, d)
    v = _normal(gen, pages, h, d, page)
    out = {"table": table.cuda(), "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda")}
    for name, x in (("k", k), ("v", v)):
        scale = _scale(x.abs().amax(dim=(2, 3)))
        out[name + "_scale"] = scale
        out[name] = (x / scale[:, :, None, None].bfloat16()).float().to(torch.float8_e4m3fn)
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    b, hk, d = case["batch"], case["kv_heads"], case["dim"]
    if case["op"] == "rope":
        s, h = case["seq"], case["heads"]

        def heads():
            if case["packed"]:
                qkv = _normal(gen, b, s, h + 2 * hk, d).permute(0, 2, 1, 3)
                return qkv[:, :h], qkv[:, h:h + hk]
            return _normal(gen, b, h, s, d), _normal(gen, b, hk, s, d)

        state = {"interleaved": case["interleaved"]}
        state["q"], state["k"] = heads()
        state["q_weight"], state["k_weight"] = (1 + 0.2 * _normal(gen, d) for _ in range(2))
        if case["train"]:   # gradients lie as the attention that gave them leaves them
            state["dq"], state["dk"] = _normal(gen, b, h, s, d), _normal(gen, b, hk, s, d)
        first = torch.randint(0, case["far"] + 1, (b, 1), generator=gen, device="cuda")
        state["positions"] = (first + torch.arange(s, device="cuda")).int()
        state["cos"], state["sin"] = _table(case["far"] + s, d)
        return {"op": "rope", "train": case["train"], **state}
    lengths, new = _lengths(case)
    state = _cache(gen, case, lengths)
    if case["op"] == "read":
        return {"op": "read", "longest": case["length"], **state}
    t = case["tokens"]
    state["counts"] = None
    if new != [t] * b:
        state["counts"] = torch.tensor(new, dtype=torch.int32, device="cuda")
    if case["op"] == "write":   # keys from their norm and rotation, values as views of the fused projection
        state["k_new"] = _normal(gen, b, hk, t, d)
        state["v_new"] = _normal(gen, b, t, 3 * hk, d).permute(0, 2, 1, 3)[:, 2 * hk:]
        return {"op": "write", **state}
    return {"op": "attend", "q": _normal(gen, b, case["heads"], t, d), **state}


def run(state):
    if own:
        return _own(state)
    return {"rope": _plain_rope, "write": _plain_write, "read": _plain_read, "attend": _plain_attend}[state["op"]](state)


_framework = None


def _own(s):
    global _framework
    if _framework is None:
        from warpir_amd import api
        _framework = api
    api = _framework
    if s["op"] == "rope":
        how = (s["q_weight"], s["k_weight"], s["cos"], s["sin"])
        out = api.qk_norm_rope(s["q"], s["k"], *how, positions=s["positions"], eps=EPS, interleaved=s["interleaved"])
        if not s["train"]:
            return out
        return (*out, *api.qk_norm_rope_backward(s["dq"], s["dk"], s["q"], s["k"], *how, positions=s["positions"],
                                                 eps=EPS, interleaved=s["interleaved"]))
    cache = api.KVCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
    if s["op"] == "write":
        return tuple(api.kv_cache_write(cache, s["k_new"], s["v_new"], s["table"], s["lengths"], counts=s["counts"]))
    if s["op"] == "read":
        return api.kv_cache_read(cache, s["table"], s["lengths"], s["longest"])
    return api.attention_cached(s["q"], cache, s["table"], s["lengths"], counts=s["counts"])


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _halves(x, interleaved):
    return (x[..., 0::2], x[..., 1::2]) if interleaved else x.chunk(2, -1)


def _whole(a, b, interleaved):
    return torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)


def _plain_rope(s):
    cos, sin = (s[n][s["positions"].long()][:, None] for n in ("cos", "sin"))   # [B, 1, S, D/2]
    inter = s["interleaved"]

    def forward(x, w):
        x = x.float()
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        a, b = _halves(y, inter)
        return _whole(a * cos - b * sin, b * cos + a * sin, inter).bfloat16()

    def backward(g, x, w):
        x, g = x.float(), g.float()
        a, b = _halves(g, inter)
        gy = _whole(a * cos + b * sin, b * cos - a * sin, inter)
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        xr = x * r
        dw = (gy * xr).sum(dim=(0, 1, 2), dtype=torch.float64).float()
        gw = gy * w.float()
        return (r * (gw - xr * (gw * xr).mean(-1, keepdim=True))).bfloat16(), dw

    out = forward(s["q"], s["q_weight"]), forward(s["k"], s["k_weight"])
    if not s["train"]:
        return out
    (dq, dqw), (dk, dkw) = backward(s["dq"], s["q"], s["q_weight"]), backward(s["dk"], s["k"], s["k_weight"])
    return (*out, dq, dk, dqw, dkw)


def _codes(x):
    return x.to(torch.float8_e4m3fn)


def _plain_write(s):
    tokens, page = s["k_new"].shape[2], s["k"].shape[2]
    lengths = s["lengths"].long()
    counts = torch.full_like(lengths, tokens) if s["counts"] is None else s["counts"].long()
    start = lengths - counts
    # the pages that can be touched, and of every place in them which new token comes there
    place = (start // page)[:, None] + torch.arange((tokens + page - 2) // page + 1, device="cuda")   # [B, N]
    touched = (place * page < lengths[:, None]) & (counts > 0)[:, None]
    place = torch.where(touched, place, (start // page)[:, None])     # others: the first one again
    at = place[:, :, None] * page + torch.arange(page, device="cuda")
    new = (at >= start[:, None, None]) & (at < lengths[:, None, None])
    old = (at < start[:, None, None])
    here = (at - start[:, None, None]).clamp(0, tokens - 1)           # [B, N, page]
    wide = place.clamp(max=s["table"].shape[1] - 1)
    ids = torch.gather(s["table"].long(), 1, wide)
    none = ((counts <= 0)[:, None] | (ids < 0)).flatten()
    ids = ids.clamp(min=0)
    # entries without a new token go nowhere: they repeat the first write of the batch
    first = torch.argsort(none.int(), stable=True)[0]
    source = torch.where(none, first, torch.arange(none.numel(), device="cuda"))
    to = ids.flatten()[source]
    rows = torch.arange(lengths.shape[0], device="cuda")[:, None, None]
    for name in ("k", "v"):
        cache, scales = s[name], s[name + "_scale"]
        x = s[name + "_new"].permute(0, 2, 1, 3)[rows, here].float().permute(0, 1, 3, 2, 4)   # [B, N, H, page, D]
        mask_new, mask_old = new[:, :, None, :, None], old[:, :, None, :, None]
        need = _scale((x.abs() * mask_new).amax(dim=(3, 4)))
        was = scales[ids]
        keeps = old.any(-1)[:, :, None] & (was >= need)
        scale = torch.where(keeps, was, need)
        held = cache.view(torch.uint8)[ids].view(cache.dtype)
        held = held if name == "k" else held.transpose(3, 4).contiguous()
        grown = (scale != was)[:, :, :, None, None] & mask_old
        again = _codes(held.float() * (was / scale)[:, :, :, None, None])
        fresh = _codes(x * (1 / scale)[:, :, :, None, None])
        bits = torch.where(mask_new, fresh.view(torch.uint8),
                           torch.where(grown, again.view(torch.uint8), held.view(torch.uint8)))
        if name == "v":
            bits = bits.transpose(3, 4)
        cache.view(torch.uint8)[to] = bits.flatten(0, 1)[source]
        scales[to] = scale.flatten(0, 1)[source]
    return s["k"], s["v"], s["k_scale"], s["v_scale"]


def _dense(s, tokens):
    """K and V of every sequence in 32 bits, [B, H, tokens, D]; places past its length hold 0."""
    page = s["k"].shape[2]
    n = -(-tokens // page)
    ids = s["table"][:, :n].long().clamp(min=0)
    seen = (torch.arange(tokens, device="cuda") < s["lengths"][:, None])[:, None, :, None]
    k = s["k"].view(torch.uint8)[ids].view(torch.float8_e4m3fn).float() * s["k_scale"][ids][..., None, None]
    k = k.permute(0, 2, 1, 3, 4).flatten(2, 3)[:, :, :tokens].masked_fill(~seen, 0)
    v = s["v"].view(torch.uint8)[ids].view(torch.float8_e4m3fn).float() * s["v_scale"][ids][..., None, None]
    v = v.permute(0, 2, 1, 4, 3).flatten(2, 3)[:, :, :tokens].masked_fill(~seen, 0)
    return k, v


def _plain_read(s):
    k, v = _dense(s, s["longest"])
    return k.bfloat16(), v.bfloat16()


def _plain_attend(s):
    q = s["q"].float()
    b, h, t, d = q.shape
    hk = s["k"].shape[1]
    n = s["table"].shape[1] * s["k"].shape[2]
    k, v = _dense(s, n)
    lengths = s["lengths"].long()
    counts = torch.full_like(lengths, t) if s["counts"] is None else s["counts"].long()
    step = torch.arange(t, device="cuda")
    pos = torch.where(step < counts[:, None], (lengths - counts)[:, None] + step, -1)   # [B, T]
    q = q.view(b, hk, h // hk * t, d)
    x = torch.matmul(q, k.transpose(2, 3)).view(b, hk, h // hk, t, n) / math.sqrt(d)
    seen = (torch.arange(n, device="cuda") <= pos[:, :, None])[:, None, None]
    x = x.masked_fill(~seen, -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(b, hk, h // hk * t, n), v).view(b, hk, h // hk, t, d)
    o = torch.where(total > 0, o / total, 0.0)
    lse = (top + torch.log(total))[..., 0]
    return o.reshape(b, h, t, d).bfloat16(), lse.reshape(b, h, t)


# ---------------------------------------------------------------------------
# work and exact values
# ---------------------------------------------------------------------------
def work(case):
    b, hk, d = case["batch"], case["kv_heads"], case["dim"]
    if case["op"] == "rope":
        rows = b * case["seq"] * (case["heads"] + hk)
        angles = 4.0 * d * min(b * case["seq"], case["far"] + case["seq"])
        passes = 10.0 if case["train"] else 4.0   # x in, y out; x and dy in, dx out
        return {"bytes": passes * rows * d + angles + 4.0 * b * case["seq"], "flops": (24.0 if case["train"] else 8.0) * rows * d}
    lengths, new = _lengths(case)
    if case["op"] == "write":
        values = 2.0 * sum(new) * hk * d
        return {"bytes": 3.0 * values + 16.0 * b, "flops": 3.0 * values}
    if case["op"] == "read":
        held = 2.0 * sum(lengths) * hk * d
        return {"bytes": held + 4.0 * b * case["length"] * hk * d, "flops": held}
    t, h = case["tokens"], case["heads"]
    pairs = sum(n * (x - n) + n * (n + 1) / 2 for x, n in zip(lengths, new))
    held = 2.0 * sum(x for x, n in zip(lengths, new) if n) * hk * d
    return {"bytes": held + 4.0 * b * h * t * d + 4.0 * b * h * t, "flops": 4.0 * h * d * pairs}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        freq = BASE ** (-torch.arange(0, case["dim"], 2, dtype=torch.float64, device="cuda") / case["dim"])
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["positions"].double()[:, None, :, None] * freq)
        half = case["dim"] // 2

        def paired(x):      # pairs as complex numbers
            x = x.double()
            return torch.complex(x[..., 0::2], x[..., 1::2]) if s["interleaved"] else torch.complex(x[..., :half], x[..., half:])

        def unpaired(z):
            z = torch.view_as_real(z)
            return z.flatten(-2) if s["interleaved"] else torch.cat((z[..., 0], z[..., 1]), -1)

        outs, grads, weights = [], [], []
        for n in "qk":
            x, w = s[n].double(), s[n + "_weight"].double()
            norm = (x.square().mean(-1, keepdim=True) + EPS).sqrt()
            outs.append(unpaired(paired(x / norm * w) * turn))
            if case["train"]:
                gy = unpaired(paired(s["d" + n]) * turn.conj())
                weights.append((gy * x / norm).sum((0, 1, 2)))
                gw = gy * w
                grads.append(gw / norm - x * (gw * x).mean(-1, keepdim=True) / norm ** 3)
        return (*outs, *grads, *weights)
    lengths, new = _lengths(case)
    page, table = case["page"], s["table"].tolist()
    if case["op"] == "write":
        if sum(-(-n // page) + 1 for n in new) > 1500:
            return None
        for i, (length, n) in enumerate(zip(lengths, new)):
            start = length - n
            for p in range(start // page, -(-length // page) if n else 0):
                lo, hi = max(start, p * page), min(length, (p + 1) * page)
                for name in "kv":
                    x = s[name + "_new"][i, :, lo - start:hi - start].double()     # [H, n, D]
                    top = x.abs().amax((1, 2)).clamp(min=1e-300)
                    e = torch.ceil(torch.log2(top / E4M3_MAX)).clamp(min=-126)
                    scale, kept = _power_of_two(e), lo - p * page
                    was = s[name + "_scale"][table[i][p]].double()
                    held = s[name][table[i][p]].double()
                    held = held if name == "k" else held.transpose(1, 2).clone()
                    if kept:
                        scale = torch.maximum(scale, was)
                        held[:, :kept] = _e4m3(held[:, :kept] * (was / scale)[:, None, None])
                    held[:, kept:kept + hi - lo] = _e4m3(x / scale[:, None, None])
                    held = (held if name == "k" else held.transpose(1, 2)).float().to(torch.float8_e4m3fn)
                    s[name].view(torch.uint8)[table[i][p]] = held.view(torch.uint8)
                    s[name + "_scale"][table[i][p]] = scale.float()
        return s["k"], s["v"], s["k_scale"].double(), s["v_scale"].double()
    longest = case["length"]

    def dense(name, i, tokens):
        """One sequence's [H, tokens, D] in 64 bits."""
        ids = [p for p in table[i][:-(-tokens // page)]]
        x = s[name].view(torch.uint8)[ids].view(torch.float8_e4m3fn).double()
        x = x if name == "k" else x.transpose(2, 3)
        x = x * s[name + "_scale"][ids].double()[:, :, None, None]
        return x.transpose(0, 1).flatten(1, 2)[:, :tokens]

    if case["op"] == "read":
        outs = []
        for name in "kv":
            out = torch.zeros(case["batch"], case["kv_heads"], longest, case["dim"], dtype=torch.float64, device="cuda")
            for i, length in enumerate(lengths):
                if length:
                    out[i, :, :length] = dense(name, i, length)
            outs.append(out)
        return outs
    b, h, t, d = s["q"].shape
    if work(case)["flops"] > 3e12:
        return None
    o = torch.zeros(b, h, t, d, dtype=torch.float64, device="cuda")
    lse = torch.full((b, h, t), -math.inf, dtype=torch.float64, device="cuda")
    for i, (length, n) in enumerate(zip(lengths, new)):
        n = min(n, t)
        if not n:
            continue
        k, v = dense("k", i, length), dense("v", i, length)
        future = torch.arange(length, device="cuda") > (length - n + torch.arange(n, device="cuda"))[:, None]
        for j in range(h):
            x = s["q"][i, j, :n].double() @ k[j // (h // case["kv_heads"])].T / math.sqrt(d)
            x = x.masked_fill(future, -math.inf)
            lse[i, j, :n] = torch.logsumexp(x, -1)
            o[i, j, :n] = torch.softmax(x, -1) @ v[j // (h // case["kv_heads"])]
    return o, lse


def _e4m3(x):
    """x rounded to the nearest e4m3 value, ties to even, by the format's definition (3 bits of fraction, exponents from -6)."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    step = _power_of_two(e - 3)
    return torch.round(x / step) * step


def _power_of_two(e):
    """2^e by its bits (pow does not give it exactly everywhere)."""
    return (e.long() + 1023 << 52).view(torch.float64)
