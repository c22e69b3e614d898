"""A packed batch of prompts on its way through a layer: the products in 8-bit
integers, the rotation by positions with several axes, and attention over
each of the packed sequences, each as a call with inputs, work and exact
values: the plain form in elementary torch operations, or (``own``) the
framework's kernels.

A case is a plain dict.  ``op`` is the call:

* ``attend``: attention over packed sequences of different lengths, causal or
  not, with grouped heads -> (O, LSE); with ``train`` its gradients too
  -> (O, LSE, dQ, dK, dV).  Rows behind the last sequence give 0 and -inf.
* ``axes``: the rotation of every query and key head by positions with up to
  four axes, of the whole head or a part -> (q, k); with ``train`` the
  gradients -> (q, k, dq, dk).
* ``quantize``: tokens in 8-bit integers with a scale each -> (codes, scales).
* ``product``: the product of such tokens with a weight in 8-bit integers with a
  scale for each channel -> bf16.

Sequence i of a packed batch is tokens ``offsets[i] .. offsets[i + 1] - 1``;
heads are ``[heads, tokens, dim]``, as views of a fused projection.
"""
import math
import random

import torch

own = False

BASE = 10000.0
SMALLEST = 2.0 ** -126


def _attend(batch, longest, heads, kv_heads, dim, **more):
    return {"op": "attend", "batch": batch, "longest": longest, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "causal": True, "train": False, "ragged": True, "padding": 0, **more}


def _axes(tokens, heads, kv_heads, dim, sections, **more):
    return {"op": "axes", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "sections": sections,
            "train": False, "interleaved": False, "packed": True, **more}


def _quantize(tokens, width, **more):
    return {"op": "quantize", "tokens": tokens, "width": width, **more}


def _product(tokens, channels, width, **more):
    return {"op": "product", "tokens": tokens, "channels": channels, "width": width, **more}


def listed():
    return [
        # a few short questions at once: the call itself is most of the time
        _attend(5, 150, 16, 4, 128, name="attend_few"),
        # the patches of a batch of images, every patch with every other of its image
        _attend(48, 1024, 16, 16, 64, causal=False, name="attend_images"),
        # the prefill of prompts of very different lengths, in a buffer with room behind them
        _attend(12, 8192, 32, 8, 128, padding=500, name="attend_prompts"),
        # a small training batch of odd lengths
        _attend(7, 700, 12, 4, 64, train=True, name="attend_train_small"),
        # a training batch of packed documents
        _attend(6, 8192, 32, 8, 128, train=True, name="attend_train"),
        # one frame's patches of a small model, half of the head turned, pairs side by side, height and width
        _axes(1369, 16, 16, 64, "8,8", interleaved=True, name="axes_image"),
        # a training batch of text, images and video: time, height and width
        _axes(32768, 32, 8, 128, "16,24,24", train=True, name="axes_train"),
        # the tokens of one decode step of a small batch
        _quantize(16, 4096, name="quantize_decode"),
        # the tokens of a large prefill
        _quantize(16384, 8192, name="quantize_prefill"),
        # a decode step: the weight's bytes
        _product(16, 6144, 4096, name="product_decode"),
        # a short packed prefill of odd length
        _product(777, 4100, 4096, name="product_odd"),
        # a large prefill
        _product(8192, 8192, 8192, name="product_prefill"),
    ]


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 100)


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _key(case):
    return case["op"], case.get("train", False)


def draw(rng):
    op = rng.choice(("attend", "attend", "axes", "quantize", "product"))
    while True:
        kv_heads = rng.choice((1, 2, 4, 8, 12, 16))
        heads = kv_heads * rng.choice((1, 2, 3, 4, 8))
        dim = rng.choice((64, 128))
        if op == "attend":
            c = _attend(_log(rng, 1, 300), _log(rng, 1, 16384), heads, kv_heads, dim, causal=rng.random() < 0.7,
                        train=rng.random() < 0.5, ragged=rng.random() < 0.8, padding=rng.choice((0, 0, rng.randint(1, 1000))))
            if c["batch"] * c["longest"] > 1 << 18:
                continue
        elif op == "axes":
            axes = rng.randint(1, 4)
            pairs = 8 * rng.randint(1, dim // 16)
            cuts = sorted(rng.randint(0, pairs) for _ in range(axes - 1))
            if rng.random() < 0.5:
                cuts = [x // 8 * 8 for x in cuts]
            parts = [y - x for x, y in zip([0] + cuts, cuts + [pairs])]
            c = _axes(_log(rng, 1, 65536), heads, kv_heads, dim, ",".join(map(str, parts)), train=rng.random() < 0.5,
                      interleaved=rng.random() < 0.4, packed=rng.random() < 0.7)
        elif op == "quantize":
            c = _quantize(_log(rng, 1, 32768), 16 * _log(rng, 1, 1024))
        else:
            c = _product(_log(rng, 1, 16384), _log(rng, 16, 16384), 16 * _log(rng, 4, 1024))
        # (the plain form's scores in 32 bits, some of them at once, have to fit beside the inputs)
        if _cost(c) <= max(_cost(x) for x in listed() if _key(x) == _key(c)) and (
                op != "attend" or heads * c["longest"] ** 2 <= 3e9):
            return c


def _lengths(case):
    """The sequences' lengths: the batch of the case, whatever the seed."""
    n, longest = case["batch"], case["longest"]
    if not case["ragged"]:
        return [longest] * n
    rng = random.Random("%d %d" % (n, longest))
    lengths = [rng.randint(1, longest) for _ in range(n)]
    lengths[n // 2] = longest
    if n > 4:   # a sequence that has no tokens
        lengths[n // 4] = 0
    return lengths


def _sections(case):
    return tuple(int(x) for x in case["sections"].split(","))


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.bfloat16)


def _codes(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda").mul_(40).round_().clamp_(-127, 127).to(torch.int8)


def _frequencies(sections):
    """Every axis has frequencies of its own, base^(-i / n) for its n pairs."""
    return torch.cat([BASE ** (-torch.arange(n, dtype=torch.float64, device="cuda") / max(n, 1)) for n in sections])


def _positions(tokens, axes):
    """Text, then frames of 24 x 32 patches, in turn: [axes, tokens]."""
    at = torch.arange(tokens, device="cuda")
    inside = at % 1024
    patch = (inside - 256).clamp(min=0)
    first = at - inside + torch.minimum(inside, torch.full_like(inside, 256))
    apart = [0 * patch, patch // 32, patch % 32, patch // 256]
    return torch.stack([first + apart[a] for a in range(axes)]).int()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op == "quantize":
        x = _normal(gen, case["tokens"], case["width"])
        return {"op": op, "x": x * (0.5 + torch.rand(case["tokens"], 1, generator=gen, device="cuda")).bfloat16()}
    if op == "product":
        m, n, k = case["tokens"], case["channels"], case["width"]
        scales = [(0.5 + torch.rand(x, generator=gen, device="cuda")) / 1000 for x in (m, n)]
        return {"op": op, "a": _codes(gen, m, k), "b": _codes(gen, n, k), "a_scale": scales[0], "b_scale": scales[1]}
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if op == "axes":
        t, sections = case["tokens"], _sections(case)

        def heads():
            if case["packed"]:
                qkv = _normal(gen, 1, t, h + 2 * hk, d).transpose(1, 2)
                return qkv[:, :h], qkv[:, h:h + hk]
            return _normal(gen, 1, h, t, d), _normal(gen, 1, hk, t, d)

        state = {"op": op, "train": case["train"], "interleaved": case["interleaved"], "sections": sections}
        state["q"], state["k"] = heads()
        if case["train"]:
            state["dq"], state["dk"] = heads()
        state["positions"] = _positions(t, len(sections))
        angle = torch.arange(t, dtype=torch.float64, device="cuda")[:, None] * _frequencies(sections)
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
        return state
    lengths = _lengths(case)
    ends = [0]
    for n in lengths:
        ends.append(ends[-1] + n)
    t = ends[-1] + case["padding"]
    qkv = _normal(gen, t, h + 2 * hk, d).transpose(0, 1)
    state = {"op": op, "train": case["train"], "causal": case["causal"], "lengths": lengths,
             "offsets": torch.tensor(ends, dtype=torch.int32, device="cuda"),
             "q": qkv[:h], "k": qkv[h:h + hk], "v": qkv[h + hk:]}
    if case["train"]:
        state["do"] = _normal(gen, t, h, d).transpose(0, 1)
    return state


def run(state):
    if own:
        return _own(state)
    return {"attend": _plain_attend, "axes": _plain_axes, "quantize": _plain_quantize,
            "product": _plain_product}[state["op"]](state)


_framework = None


def _own(s):
    global _framework
    if _framework is None:
        from warpir_amd import api
        _framework = api
    api = _framework
    if s["op"] == "attend":
        o, lse = api.attention_packed(s["q"], s["k"], s["v"], s["offsets"], causal=s["causal"])
        if not s["train"]:
            return o, lse
        return (o, lse, *api.attention_packed_backward(s["q"], s["k"], s["v"], o, lse, s["do"], s["offsets"],
                                                       causal=s["causal"]))
    if s["op"] == "axes":
        how = (s["cos"], s["sin"], s["positions"], s["sections"])
        out = api.rope_axes(s["q"], s["k"], *how, interleaved=s["interleaved"])
        if not s["train"]:
            return out
        return (*out, *api.rope_axes_backward(s["dq"], s["dk"], *how, interleaved=s["interleaved"]))
    if s["op"] == "quantize":
        return api.quantize_int8(s["x"])
    return api.gemm_int8(s["a"], s["b"], s["a_scale"], s["b_scale"])


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _plain_attend(s):
    q, k, v = s["q"], s["k"], s["v"]
    h, t, d = q.shape
    hk = k.shape[0]
    g = h // hk
    o = torch.zeros(t, h, d, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    lse = torch.full((h, t), -math.inf, device="cuda")
    grads = [torch.zeros(t, x.shape[0], d, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
             for x in (q, k, v)] if s["train"] else []
    at = 0
    for n in s["lengths"]:
        rows = slice(at, at + n)
        at += n
        if n == 0:
            continue
        qs, ks, vs = (x[:, rows].float() for x in (q, k, v))
        qs, ks, vs = qs.reshape(hk, g, n, d), ks[:, None], vs[:, None]
        x = torch.matmul(qs, ks.transpose(2, 3)) / math.sqrt(d)
        if s["causal"]:
            x = x.masked_fill(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), -math.inf)
        top = x.amax(-1, keepdim=True)
        p = torch.exp(x - top)
        del x
        total = p.sum(-1, keepdim=True)
        p /= total
        out = torch.matmul(p, vs)
        o[:, rows] = out.reshape(h, n, d).bfloat16()
        lse[:, rows] = (top + torch.log(total)).reshape(h, n)
        if s["train"]:
            do = s["do"][:, rows].float().reshape(hk, g, n, d)
            # the forward's output as it was stored
            dots = (do * o[:, rows].float().reshape(hk, g, n, d)).sum(-1, keepdim=True)
            ds = p * (torch.matmul(do, vs.transpose(2, 3)) - dots) / math.sqrt(d)
            grads[0][:, rows] = torch.matmul(ds, ks).reshape(h, n, d).bfloat16()
            grads[1][:, rows] = torch.matmul(ds.transpose(2, 3), qs).sum(1).bfloat16()
            grads[2][:, rows] = torch.matmul(p.transpose(2, 3), do).sum(1).bfloat16()
    return (o, lse, *grads)


def _plain_axes(s):
    starts = [0]
    for n in s["sections"]:
        starts.append(starts[-1] + n)
    pairs = starts[-1]
    cos, sin = (torch.cat([s[name][s["positions"][a].long(), starts[a]:starts[a + 1]]
                           for a in range(len(s["sections"]))], -1) for name in ("cos", "sin"))   # [T, pairs]

    def turn(x, sign):
        y = x.float()
        part, rest = y[..., :2 * pairs], y[..., 2 * pairs:]
        if s["interleaved"]:
            a, b = part[..., 0::2], part[..., 1::2]
        else:
            a, b = part[..., :pairs], part[..., pairs:]
        first, second = a * cos - sign * b * sin, b * cos + sign * a * sin
        if s["interleaved"]:
            part = torch.stack((first, second), -1).flatten(-2)
        else:
            part = torch.cat((first, second), -1)
        return torch.cat((part, rest), -1).bfloat16()

    out = turn(s["q"], 1), turn(s["k"], 1)
    return (*out, turn(s["dq"], -1), turn(s["dk"], -1)) if s["train"] else out


def _plain_quantize(s):
    x = s["x"].float()
    scale = (x.abs().amax(1) / 127).clamp(min=SMALLEST)
    # (a quotient next to a border between two codes needs more than 32 bits)
    return torch.round(s["x"].double() / scale.double()[:, None]).to(torch.int8), scale


def _plain_product(s):
    a, b = s["a"], s["b"]
    total = torch.zeros(a.shape[0], b.shape[0], dtype=torch.int32, device="cuda")
    for k in range(0, a.shape[1], 1024):   # 1024 products of 128 * 127 at most add up to less than 2^24: exact in 32 bits
        total += torch.matmul(a[:, k:k + 1024].float(), b[:, k:k + 1024].float().T).int()
    return (total.float() * s["a_scale"][:, None] * s["b_scale"]).bfloat16()


# ---------------------------------------------------------------------------
# work and exact values
# ---------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "quantize":
        return {"bytes": 3.0 * case["tokens"] * case["width"] + 4.0 * case["tokens"],
                "flops": 2.0 * case["tokens"] * case["width"]}
    if op == "product":
        m, n, k = case["tokens"], case["channels"], case["width"]
        return {"bytes": (m + n) * (k + 4.0) + 2.0 * m * n, "flops": 2.0 * m * n * k}
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if op == "axes":
        t, sections = case["tokens"], _sections(case)
        turns = 2 if case["train"] else 1
        return {"bytes": turns * 4.0 * t * (h + hk) * d + 8.0 * t * sum(sections) + 4.0 * t * len(sections),
                "flops": turns * 6.0 * t * (h + hk) * sum(sections)}
    lengths = _lengths(case)
    t = sum(lengths)
    pairs = sum(n * (n + 1) / 2 if case["causal"] else n * n for n in lengths)
    size, flops = 4.0 * t * (h + hk) * d + 4.0 * h * t, 4.0 * h * d * pairs
    if case["train"]:   # Q, O, dO, K, V and LSE in, dQ, dK, dV out; five products of the forward's two's kind
        size, flops = size + 8.0 * t * (h + hk) * d + 4.0 * h * t, 14.0 * h * d * pairs
    return {"bytes": size, "flops": flops}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        top = s["x"].double().abs().max(1).values
        scale = (top / 127).float().double().clamp(min=SMALLEST)   # the scale as it is held
        ratio = s["x"].double().abs() / scale[:, None]
        whole = ratio.floor()
        rest = ratio - whole
        code = whole + ((rest > 0.5) | ((rest == 0.5) & (whole % 2 == 1))).double()
        return (code * s["x"].double().sign()).to(torch.int8), top.div(127).clamp(min=SMALLEST)
    if op == "product":
        out = s["a"].double() @ s["b"].double().T
        return out.mul_(s["b_scale"].double()).mul_(s["a_scale"].double()[:, None])
    if op == "axes":
        sections, t = s["sections"], case["tokens"]
        axis = [a for a, n in enumerate(sections) for _ in range(n)]
        angle = s["positions"][axis].double().T * _frequencies(sections)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), angle)
        pairs = len(axis)

        def rotated(x, by):
            x = x.double().clone()
            part = x[..., :2 * pairs]
            if s["interleaved"]:
                z = torch.view_as_complex(part.unflatten(-1, (pairs, 2)).contiguous()) * by
                x[..., :2 * pairs] = torch.view_as_real(z).flatten(-2)
            else:
                z = torch.complex(part[..., :pairs].contiguous(), part[..., pairs:].contiguous()) * by
                x[..., :pairs], x[..., pairs:2 * pairs] = z.real, z.imag
            return x

        out = [rotated(s["q"], turn), rotated(s["k"], turn)]
        return out + [rotated(s["dq"], turn.conj()), rotated(s["dk"], turn.conj())] if case["train"] else out
    h, t, d = s["q"].shape
    if work(case)["flops"] > 3e13 or h * case["batch"] > 15000:
        return None
    o = torch.zeros(h, t, d, dtype=torch.float64, device="cuda")
    lse = torch.full((h, t), -math.inf, dtype=torch.float64, device="cuda")
    grads = [torch.zeros(x.shape, dtype=torch.float64, device="cuda") for x in (s["q"], s["k"], s["v"])]
    at = 0
    for n in s["lengths"]:
        rows = slice(at, at + n)
        at += n
        if n == 0:
            continue
        future = torch.arange(n, device="cuda") > torch.arange(n, device="cuda")[:, None]
        for i in range(h):
            j = i * case["kv_heads"] // h
            q, k, v = s["q"][i, rows].double(), s["k"][j, rows].double(), s["v"][j, rows].double()
            x = q @ k.T / math.sqrt(d)
            if case["causal"]:
                x[future] = -math.inf
            lse[i, rows] = torch.logsumexp(x, -1)
            p = torch.softmax(x, -1)
            del x
            out = o[i, rows] = p @ v
            if case["train"]:
                do = s["do"][i, rows].double()
                grads[2][j, rows] += p.T @ do
                dp = do @ v.T
                p *= dp - (do * out).sum(-1, keepdim=True)
                grads[0][i, rows] = p @ k / math.sqrt(d)
                grads[1][j, rows] += p.T @ q / math.sqrt(d)
    return (o, lse, *grads) if case["train"] else (o, lse)
