"""The 64-bit oracles of the layer operators against differences and direct
sums, on the CPU."""
import math

import pytest
import torch

from oracle.layer_ref import (angles_ref, attention_cached_ref, cache_read_ref, cache_write_ref, e4m3_ref,
                              norm_rope_bwd_ref, norm_rope_ref, scale_ref)


@pytest.mark.parametrize("interleaved", [False, True])
def test_norm_rope_gradient_against_differences(interleaved):
    gen = torch.Generator().manual_seed(0)
    x, g = (torch.randn(2, 3, 4, 8, generator=gen, dtype=torch.float64) for _ in range(2))
    w = torch.rand(8, generator=gen, dtype=torch.float64) + 0.5
    angle = angles_ref(torch.randint(0, 50, (2, 4), generator=gen), 8)

    def loss(x, w):
        return (norm_rope_ref(x, w, angle, 1e-3, interleaved)[0] * g).sum()

    dx, dw, _, _ = norm_rope_bwd_ref(g, x, w, angle, 1e-3, interleaved)
    h = 1e-6
    for at in ((0, 0, 0, 0), (1, 2, 3, 7), (0, 1, 2, 4), (1, 0, 1, 3)):
        step = torch.zeros_like(x)
        step[at] = h
        assert abs((loss(x + step, w) - loss(x - step, w)) / (2 * h) - dx[at]) < 1e-7
    for i in range(8):
        step = torch.zeros_like(w)
        step[i] = h
        assert abs((loss(x, w + step) - loss(x, w - step)) / (2 * h) - dw[i]) < 1e-7


def test_rotation_keeps_relative_positions():
    """Scores of rotated rows depend on the distance alone."""
    q, k = (torch.randn(1, 1, 1, 16, dtype=torch.float64).expand(1, 1, 6, 16) for _ in range(2))
    w = torch.ones(16)
    for inter in (False, True):
        a = norm_rope_ref(q, w, angles_ref(torch.arange(6)[None], 16), 0.0, inter)[0]
        b = norm_rope_ref(k, w, angles_ref(torch.arange(6)[None] + 4, 16), 0.0, inter)[0]
        s = (a * b).sum(-1)
        assert torch.allclose(s, s[..., :1].expand_as(s))


def test_e4m3_and_scales():
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    fine = every[every.isfinite()].unique()
    assert torch.equal(e4m3_ref(fine).double(), fine)
    mid = (fine[1:] + fine[:-1]) / 2
    assert torch.equal(e4m3_ref(mid).double(), mid.float().to(torch.float8_e4m3fn).double())   # ties to even
    assert bool(((e4m3_ref(mid + 1e-9).double() - fine[1:]).abs() < 1e-12).all())
    assert scale_ref(448.0) == 1.0 and scale_ref(448.1) == 2.0 and scale_ref(0.0) == 2.0 ** -126
    assert scale_ref(2.0 ** -9 * 1.75 * 256) == 2.0 ** -9


def test_cache_and_attention_against_dense():
    gen = torch.Generator().manual_seed(3)
    cache = (torch.zeros(5, 2, 16, 64, dtype=torch.uint8).view(torch.float8_e4m3fn),
             torch.zeros(5, 2, 64, 16, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros(5, 2), torch.zeros(5, 2))
    table = torch.tensor([[3, 1, -1], [0, 4, 2]], dtype=torch.int32)
    k, v = (torch.randn(2, 2, 30, 64, generator=gen).bfloat16() for _ in range(2))
    cache_write_ref(cache, k, v, table, [30, 20], [30, 20])
    kr, vr, there = cache_read_ref(cache, table, [30, 20], 32)
    assert bool(there[0, :30].all()) and not bool(there[0, 30:].any()) and there[1].sum() == 20
    for got, want in ((kr, k), (vr, v)):   # half a step of e4m3, or of its subnormals at the page's scale
        off = (got[0, :, :30] - want[0].double()).abs()
        assert bool((off <= 2.0 ** -4 * want[0].double().abs() + 2.0 ** -10 * cache[2].max()).all())
    q = torch.randn(2, 4, 3, 64, generator=gen)
    o, lse, _ = attention_cached_ref(q, cache, table, [30, 20], [3, 1])
    s = torch.einsum("htd,hnd->htn", q[0].double(), kr[0, :, :30].repeat_interleave(2, 0)) / 8
    s = s.masked_fill(torch.arange(30) > 27 + torch.arange(3)[:, None], -math.inf)
    assert torch.allclose(lse[0], torch.logsumexp(s, -1))
    assert torch.allclose(o[0], torch.softmax(s, -1) @ vr[0, :, :30].repeat_interleave(2, 0))
    assert bool((o[1, :, 1:] == 0).all()) and bool((lse[1, :, 1:] == -math.inf).all())
