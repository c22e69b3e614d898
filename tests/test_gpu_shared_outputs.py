"""Destinations that are an input: the results of a call with memory of its
own; and those that would be read while they are written: refused."""
import pytest
import torch

from oracle.torch_ref import seeded_normal
from tests.conftest import announce
from warpir_amd import api, kvcache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,hkv,tokens,columns,forced", [
    (8, 2, 1, 12, None), (8, 2, 1, 200, None), (8, 2, 7, 12, None), (8, 2, 300, 12, None),
    (6, 2, 50, 12, (16, 4, 0, 0)), (6, 2, 50, 12, (16, 4, 40, 1)), (6, 2, 50, 12, (32, 4, 0, 0)),
    (6, 2, 50, 12, (128, 4, 0, 0)), (6, 2, 50, 12, (128, 8, 0, 0)), (6, 2, 50, 12, (128, 4, 40, 1))])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_over_its_queries(gpu, monkeypatch, heads, hkv, tokens, columns, forced, d):
    announce(f"attention cached in place H{heads}/{hkv} T{tokens} D{d} {columns} pages {forced}")
    if forced:
        monkeypatch.setattr(kvcache, "_attention_form", lambda *a: forced)
        monkeypatch.setattr(kvcache, "_attention_plans", kvcache.DevicePlans("attention_cached"))
    cache = api.KVCache.empty(3 * columns, hkv, 32, d)
    table = torch.arange(3 * columns, dtype=torch.int32, device="cuda").view(3, columns)
    lengths = torch.tensor([columns * 32, tokens, columns * 17], dtype=torch.int32, device="cuda")
    counts = torch.tensor([tokens, tokens // 2, tokens], dtype=torch.int32, device="cuda")
    k, v = (seeded_normal((3, hkv, columns * 32, d), s).cuda() for s in (1, 2))
    api.kv_cache_write(cache, k, v, table, lengths, lengths)
    wide = seeded_normal((3, tokens, heads + 2, d), 3).cuda().permute(0, 2, 1, 3)
    want = api.attention_cached(wide[:, 1:heads + 1], cache, table, lengths, counts)
    for _ in range(2):
        x = wide.clone()
        q = x[:, 1:heads + 1]
        got = api.attention_cached(q, cache, table, lengths, counts, out=q)
        assert got[0] is q and torch.equal(q, want[0]) and torch.equal(got[1], want[1])
        assert torch.equal(x[:, [0, heads + 1]], wide[:, [0, heads + 1]])
    with pytest.raises(ValueError, match="out and q have memory in common"):
        api.attention_cached(x[:, 1:heads + 1], cache, table, lengths, counts, out=x[:, :heads])


def test_norm_rope_over_the_other_input_is_refused(gpu):
    qkv = seeded_normal((2, 19, 12, 64), 1).cuda().permute(0, 2, 1, 3)
    q, k, w = qkv[:, :4], qkv[:, 4:8], torch.ones(64, dtype=torch.bfloat16, device="cuda")
    table = api.rope_table(32, 64)
    want = api.qk_norm_rope(q, k, w, w, *table)
    for outs in ((k, q), (k, None), (None, q), (qkv[:, 1:5], qkv[:, 8:]), (qkv[:, 8:], qkv[:, 8:])):
        with pytest.raises(ValueError, match="have memory in common"):
            api.qk_norm_rope(q, k, w, w, *table, q_out=outs[0], k_out=outs[1])
    free = qkv.clone()
    got = api.qk_norm_rope(q, k, w, w, *table, q_out=free[:, :4], k_out=free[:, 4:8])
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    got = api.qk_norm_rope(q, k, w, w, *table, q_out=qkv[:, 8:], k_out=k)   # one that is free, one in place
    assert got[1] is k and all(torch.equal(x, y) for x, y in zip(got, want))
