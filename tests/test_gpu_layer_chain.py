"""The operators one after another, as a layer uses them: every stage against
its oracle on what the stage before it gave, with that stage's tolerance."""
import math

import pytest
import torch

from oracle.layer_ref import (angles_ref, attention_cached_ref, cache_read_ref, cache_write_ref, norm_rope_bwd_ref,
                              norm_rope_ref)
from oracle.torch_ref import attention_bwd_ref, attention_ref, gemm_ref, rel_err, seeded_normal
from tests.conftest import announce
from warpir_amd import api, kvcache

pytestmark = pytest.mark.gpu


def _heads(qkv, b, s, h, hk, d):
    """q, k, v of a fused projection's [B * S, (H + 2 H_kv) * D] output, as views."""
    x = qkv.view(b, s, h + 2 * hk, d).permute(0, 2, 1, 3)
    return x[:, :h], x[:, h:h + hk], x[:, h + hk:]


def _near_rope(got, x, w, angle):
    ref, size = norm_rope_ref(x.cpu(), w.cpu(), angle)
    assert bool(((got.cpu().double() - ref).abs() <= 2 ** -8 * ref.abs() + 2 ** -18 * size).all())


@pytest.mark.parametrize("d,h,hk", [(64, 4, 4), (128, 4, 2)])
def test_training_layer(gpu, d, h, hk):
    """x -> projection -> norm and rotation -> causal attention -> projection, and back to the weights."""
    announce(f"training layer H{h}/{hk} D{d}")
    b, s, width = 2, 192, 256
    x = seeded_normal((b * s, width), 0).cuda()
    wqkv = (seeded_normal((width, (h + 2 * hk) * d), 1).float() / math.sqrt(width)).bfloat16().cuda()
    wo = (seeded_normal((h * d, width), 2).float() / math.sqrt(h * d)).bfloat16().cuda()
    qw, kw = ((1 + 0.2 * seeded_normal((d,), 3 + i).float()).bfloat16().cuda() for i in range(2))
    table = api.rope_table(s, d)
    angle = angles_ref(torch.arange(s)[None], d)

    qkv = api.gemm(x, wqkv)
    assert rel_err(qkv.cpu(), gemm_ref(x.cpu(), wqkv.cpu())) <= 1e-2
    q, k, v = _heads(qkv, b, s, h, hk, d)
    qr, kr = api.qk_norm_rope(q, k, qw, kw, *table)
    _near_rope(qr, q, qw, angle), _near_rope(kr, k, kw, angle)
    o, lse = api.attention_forward(qr, kr, v, causal=True)
    group = h // hk
    kv = [t.cpu().repeat_interleave(group, 1) for t in (kr, v)]
    assert rel_err(o.cpu(), attention_ref(qr.cpu(), *kv, scale=1 / math.sqrt(d), causal=True)[0]) <= 1e-2
    flat = o.transpose(1, 2).reshape(b * s, h * d)
    y = api.gemm(flat, wo)
    assert rel_err(y.cpu(), gemm_ref(flat.cpu(), wo.cpu())) <= 1e-2

    dy = seeded_normal(y.shape, 9).cuda()
    do = api.gemm(dy, wo.t().contiguous()).view(b, s, h, d).transpose(1, 2)
    dqr, dkr, dv = api.attention_backward(qr, kr, v, o, lse, do, causal=True, dv=torch.empty(v.shape, dtype=v.dtype, device="cuda"))
    ref = attention_bwd_ref(qr.cpu(), *kv, do.cpu(), scale=1 / math.sqrt(d), causal=True)
    for got, want, shared in ((dqr, ref[0], 1), (dkr, ref[1], group), (dv, ref[2], group)):
        want = want.view(b, -1, shared, s, d).sum(2)
        assert rel_err(got.cpu(), want) <= 1e-2
    # the projection's gradient in its own layout: dq and dk are written where they belong
    dqkv = torch.empty_like(qkv)
    dq, dk, dvv = _heads(dqkv, b, s, h, hk, d)
    got = api.qk_norm_rope_backward(dqr, dkr, q, k, qw, kw, *table, dq=dq, dk=dk)
    dvv.copy_(dv)
    for dx, dw, g, t, w in ((dq, got[2], dqr, q, qw), (dk, got[3], dkr, k, kw)):
        want, want_w, size, size_w = norm_rope_bwd_ref(g.cpu(), t.cpu(), w.cpu(), angle)
        assert bool(((dx.cpu().double() - want).abs() <= 2 ** -8 * want.abs() + 2 ** -17 * size).all())
        assert bool(((dw.cpu().double() - want_w).abs() <= 2 ** -15 * size_w).all())
    dwqkv = api.gemm(x.t().contiguous(), dqkv)
    assert rel_err(dwqkv.cpu(), gemm_ref(x.cpu().t(), dqkv.cpu())) <= 1e-2


@pytest.mark.parametrize("d,h,hk,page", [(64, 4, 2, 16), (128, 8, 2, 64)])
def test_serving_layer(gpu, d, h, hk, page):
    """Prompts of unequal length, then single tokens and a few drafted ones: projection -> norm and rotation -> cache ->
    attention over it, with a copy of the cache that the oracle keeps."""
    announce(f"serving layer H{h}/{hk} D{d} page {page}")
    b, width, columns = 3, 128, -(-150 // page)
    w = (seeded_normal((width, (h + 2 * hk) * d), 1).float() / math.sqrt(width)).bfloat16().cuda()
    qw, kw = ((1 + 0.2 * seeded_normal((d,), 3 + i).float()).bfloat16().cuda() for i in range(2))
    cos, sin = api.rope_table(256, d)
    cache = api.KVCache.empty(b * columns, hk, page, d)
    kept = [t.cpu().clone() for t in cache]
    table = torch.randperm(b * columns, generator=torch.Generator().manual_seed(0)).view(b, columns).int()
    lengths = torch.zeros(b, dtype=torch.int32)
    for step, (tokens, counts) in enumerate([(70, (70, 33, 1)), (1, (1, 1, 1)), (4, (4, 2, 4)), (1, (1, 0, 1)), (40, (17, 40, 0))]):
        counts = torch.tensor(counts, dtype=torch.int32)
        lengths = lengths + counts
        where = (lengths - counts)[:, None] + torch.arange(tokens)
        x = seeded_normal((b * tokens, width), 10 + step).cuda()
        q, k, v = _heads(api.gemm(x, w), b, tokens, h, hk, d)
        q2, k2 = api.qk_norm_rope(q, k, qw, kw, cos, sin, positions=where.int().cuda())
        _near_rope(q2, q, qw, angles_ref(where, d)), _near_rope(k2, k, kw, angles_ref(where, d))
        on = dict(page_table=table.cuda(), lengths=lengths.cuda(), counts=counts.cuda())
        api.kv_cache_write(cache, k2, v, **on)
        cache_write_ref(kept, k2.cpu(), v.cpu(), table, lengths, counts)
        assert all(torch.equal(a.cpu().float(), c.float()) for a, c in zip(cache, kept))
        o, lse = api.attention_cached(q2, cache, **on)
        ref, ref_lse, weight = attention_cached_ref(q2.cpu(), kept, table, lengths, counts)
        assert bool(((o.cpu().double() - ref).abs() <= 2 ** -8 * ref.abs() + (2 ** -8 + 2 ** -12) * weight).all())
        seen = ref_lse.isfinite()
        assert torch.equal(lse.cpu().isfinite(), seen) and (lse.cpu().double() - ref_lse)[seen].abs().max() <= 2 ** -11
    dense = api.kv_cache_read(cache, table.cuda(), lengths.cuda(), 150)
    want = cache_read_ref(kept, table, lengths, 150)
    assert torch.equal(dense[0].cpu().double(), want[0]) and torch.equal(dense[1].cpu().double(), want[1])


def test_cached_attention_is_the_dense_one_on_what_the_cache_holds(gpu):
    """A prompt's attention over the cache against api.attention_forward on the keys and values read back."""
    b, h, hk, s, d = 2, 8, 2, 256, 128
    cache = api.KVCache.empty(16, hk, 64, d)
    table = torch.arange(8, dtype=torch.int32).view(2, 4).cuda()
    lengths = torch.full((2,), s, dtype=torch.int32, device="cuda")
    q = seeded_normal((b, h, s, d), 0).cuda()
    k, v = (seeded_normal((b, hk, s, d), i).cuda() for i in (1, 2))
    api.kv_cache_write(cache, k, v, table, lengths)
    o, lse = api.attention_cached(q, cache, table, lengths)
    kd, vd = api.kv_cache_read(cache, table, lengths, s)
    od, lsed = api.attention_forward(q, kd, vd, causal=True)
    # both round the probabilities and O to bf16 (2^-8 of sum p |v|, which is under max |v|, and of O)
    assert float((o.float() - od.float()).abs().max()) <= 4 * 2 ** -8 * float(vd.abs().max())
    assert float((lse - lsed).abs().max()) <= 2 ** -11


def test_one_tensor_for_lengths_and_counts(gpu):
    """Whole prompts: the results and the plans of two tensors."""
    n = torch.tensor((90, 1, 37), dtype=torch.int32, device="cuda")
    q, k, v = (seeded_normal((3, h, 90, 64), i).cuda() for i, h in enumerate((4, 2, 2)))
    table = torch.arange(9, dtype=torch.int32, device="cuda").view(3, 3)
    got = []
    for counts in (n.clone(), n, n):
        cache = api.KVCache.empty(9, 2, 32, 64)
        api.kv_cache_write(cache, k, v, table, n, counts)
        got.append((*(x.view(torch.uint8) for x in cache), *api.attention_cached(q, cache, table, n, counts)))
    assert all(torch.equal(x, y) for other in got[1:] for x, y in zip(got[0], other))
    assert kvcache._write_plans.run(0, k, v, *cache, table, n, n.view_as(n)) is not False
