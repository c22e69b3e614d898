"""The 64-bit oracles of the packed operators against autograd, differences and
direct sums, and the numbering of the packed blocks, on the CPU."""
import math
import random

import pytest
import torch

from oracle.packed_ref import (axes_angles_ref, gemm_int8_ref, packed_attention_bwd_ref, packed_attention_ref,
                               quantize_ref, rope_axes_ref)


def _inputs(h, hk, offsets, d, rest=3):
    gen = torch.Generator().manual_seed(1)
    t = offsets[-1] + rest
    return [torch.randn(n, t, d, generator=gen, dtype=torch.float64) for n in (h, hk, hk, h)]


@pytest.mark.parametrize("causal", [False, True])
def test_attention_row_by_row(causal):
    offsets = [0, 3, 3, 4, 9]
    q, k, v, _ = _inputs(4, 2, offsets, 8)
    o, lse, _, _ = packed_attention_ref(q, k, v, offsets, causal)
    for a, b in zip(offsets, offsets[1:]):
        for p in range(a, b):
            seen = range(a, p + 1 if causal else b)
            for i in range(4):
                w = [math.exp(float(q[i, p] @ k[i // 2, j]) / math.sqrt(8)) for j in seen]
                want = sum(x * v[i // 2, j] for x, j in zip(w, seen)) / sum(w)
                assert torch.allclose(o[i, p], want, rtol=1e-12, atol=1e-12)
                assert abs(float(lse[i, p]) - math.log(sum(w))) < 1e-12
    assert bool((o[:, 9:] == 0).all()) and bool((lse[:, 9:] == -math.inf).all())


@pytest.mark.parametrize("causal", [False, True])
def test_gradients_against_differences(causal):
    offsets = [0, 5, 6, 6, 10]
    q, k, v, do = _inputs(4, 2, offsets, 4)
    o, lse, _, _ = packed_attention_ref(q, k, v, offsets, causal)
    grads = packed_attention_bwd_ref(q, k, v, o, lse, do, offsets, causal)[0]

    def loss(x):
        return float((packed_attention_ref(*x, offsets, causal)[0] * do).sum())

    rng, step = random.Random(0), 1e-5
    for which, grad in enumerate(grads):
        for _ in range(12):
            at = tuple(rng.randrange(n) for n in grad.shape)
            up, down = [q.clone(), k.clone(), v.clone()], [q.clone(), k.clone(), v.clone()]
            up[which][at] += step
            down[which][at] -= step
            assert abs((loss(up) - loss(down)) / (2 * step) - float(grad[at])) < 1e-7


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation(interleaved):
    """Turning back undoes it, lengths of pairs stay, and the gradient is the rotation back."""
    gen = torch.Generator().manual_seed(0)
    x, g = (torch.randn(2, 3, 5, 24, generator=gen, dtype=torch.float64) for _ in "xg")
    freq = torch.rand(8, generator=gen, dtype=torch.float64)
    pos = torch.randint(0, 40, (3, 2, 5), generator=gen)
    angle = axes_angles_ref(pos, freq, (3, 0, 5))
    assert float(angle[1, 2, 3]) == float(pos[2, 1, 2] * freq[3])
    out, _ = rope_axes_ref(x, angle, interleaved)
    assert torch.equal(out[..., 16:], x[..., 16:]) and not torch.allclose(out[..., :16], x[..., :16])
    assert torch.allclose(rope_axes_ref(out, angle, interleaved, back=True)[0], x)
    back, _ = rope_axes_ref(g, angle, interleaved, back=True)
    leaf = x.clone().requires_grad_()
    (rope_axes_ref(leaf, angle, interleaved)[0] * g).sum().backward()
    assert torch.allclose(leaf.grad, back)


def test_integer_rows():
    x = torch.tensor([[127.0, 0.5, 1.5, -2.5, -126.5, 0.0], [0.0] * 6, [1.0, math.inf, 0, 0, 0, 0]])
    codes, scale = quantize_ref(x)
    assert codes[0].tolist() == [127, 0, 2, -2, -126, 0] and float(scale[0]) == 1.0
    assert codes[1].tolist() == [0] * 6 and float(scale[1]) == 2.0 ** -126
    assert math.isnan(float(scale[2])) and codes[2].tolist() == [0] * 6
    out = gemm_int8_ref(codes[:1], codes[:1], scale[:1], scale[:1])
    assert float(out[0, 0]) == 127 ** 2 + 2 ** 2 + 2 ** 2 + 126 ** 2


def _block(offsets, batch, tokens, x, rows=128):
    """(sequence, start, length, first row) as wir_packed.h's packed_block finds them, 64 sequences at a time."""
    def at(i):
        return tokens if i > batch else min(max(offsets[i], 0), tokens)

    lo, n = 0, batch + 1
    while True:
        step = -(-n // 64)
        here = [i for i in range(64) if i * step < n and at(min(lo + i * step, batch)) // rows + lo + i * step <= x]
        last = max(here, default=0)
        if step == 1:
            break
        lo, n = lo + last * step, min(step, n - last * step)
    start = at(min(lo + last, batch))
    return lo + last, start, at(min(lo + last, batch) + 1) - start, (x - start // rows - lo - last) * rows


@pytest.mark.parametrize("batch", [0, 1, 2, 5, 62, 63, 64, 65, 130, 4095, 4096, 5000])
def test_numbers_of_packed_blocks(batch):
    """Every block of every sequence, and of the tokens behind them, has one number; whatever the
    offsets, no block leaves the tokens."""
    for seed in range(2 if batch > 1000 else 8):
        rng = random.Random(seed)
        lengths = [rng.choice((0, 0, 1, 127, 128, 129, rng.randint(0, 700))) for _ in range(batch)]
        offsets = [0]
        for n in lengths:
            offsets.append(offsets[-1] + n)
        tokens = offsets[-1] + rng.choice((0, 1, 128, 300))
        numbers = tokens // 128 + batch + 1
        found = [_block(offsets, batch, tokens, x) for x in range(numbers)]
        got = [(i, row) for i, _, n, row in found if 0 <= row < n]
        want = [(i, row) for i, n in enumerate(lengths + [tokens - offsets[-1]]) for row in range(0, n, 128)]
        assert sorted(got) == want
        wild = [rng.randint(-300, tokens + 300) for _ in offsets]
        for x in range(numbers):
            _, start, n, row = _block(wild, batch, tokens, x)
            assert not 0 <= row < n or (0 <= start and start + n <= tokens)
