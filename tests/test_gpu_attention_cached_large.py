"""Attention over the paged 8-bit cache with 2^24 query rows and more in one
call: every sequence is as in a call of a few."""
import pytest
import torch

from tests.conftest import announce
from warpir_amd import api, kvcache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch,heads,hkv,tokens,columns,few", [(64, 64, 8, 4096, 66, 8), (300, 64, 8, 1000, 18, 20)])
def test_many_prompts(gpu, batch, heads, hkv, tokens, columns, few):
    d, page = 64, 64
    assert batch * heads * tokens >= 1 << 24
    form = kvcache._attention_form(tokens * heads // hkv, batch * hkv, columns, page, d)
    assert form[2] == 0 and form == kvcache._attention_form(tokens * heads // hkv, few * hkv, columns, page, d)
    announce(f"attention cached B{batch} H{heads}/{hkv} T{tokens} of D{d}, {batch * heads * tokens} query rows, form {form}")
    gen = torch.Generator(device="cuda").manual_seed(3)
    cache = api.KVCache.empty(columns, hkv, page, d)
    first = torch.arange(columns, dtype=torch.int32, device="cuda")[None]
    k, v = (torch.randn(1, hkv, columns * page, d, generator=gen, device="cuda").bfloat16() for _ in "kv")
    api.kv_cache_write(cache, k, v, first, torch.tensor([columns * page], dtype=torch.int32, device="cuda"))
    table = torch.stack([torch.roll(first[0], i) for i in range(batch)])   # pages that are read may be shared
    lengths = torch.tensor([tokens + i % (columns * page - tokens) for i in range(batch)], dtype=torch.int32, device="cuda")
    q = torch.randn(batch, heads, tokens, d, generator=gen, device="cuda", dtype=torch.bfloat16)
    o, lse = api.attention_cached(q, cache, table, lengths)
    for at in (0, batch // 2, batch - few):
        some = slice(at, at + few)
        want = api.attention_cached(q[some], cache, table[some].contiguous(), lengths[some])
        assert torch.equal(o[some], want[0]) and torch.equal(lse[some], want[1])
        assert bool(lse[some].isfinite().all())
