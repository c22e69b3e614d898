"""Destinations that share memory with another tensor of the call: which
layouts do, against counting bytes, and the calls that refuse them."""
import os
import random

import pytest
import torch

from warpir_amd import api, handwritten, plans
from warpir_amd.runtime import PKG_DIR

pytestmark = pytest.mark.skipif(not os.path.exists(os.path.join(PKG_DIR, "_wir_plans.so")), reason="not built")


def _bytes(t):
    at = torch.zeros(t.shape, dtype=torch.int64)
    for d, (n, s) in enumerate(zip(t.shape, t.stride())):
        at += (torch.arange(n) * s * t.element_size()).view([-1 if i == d else 1 for i in range(t.dim())])
    return {t.data_ptr() + int(x) + i for x in at.flatten() for i in range(t.element_size())}


def test_against_counting():
    rng = random.Random(5)
    buf = torch.zeros(4000, dtype=torch.bfloat16)
    mod, found = plans.native(), [0, 0]
    for _ in range(4000):
        pair = []
        for _ in range(2):
            dtype = rng.choice((torch.bfloat16, torch.bfloat16, torch.float32))
            b = buf.view(dtype)
            shape = [rng.randint(1, 4) for _ in range(rng.randint(1, 4))]
            stride = [rng.choice((0, 1, 1, 2, 3, 4, 8, 8, 24, 96)) for _ in shape]
            pair.append(b.as_strided(shape, stride, rng.randint(0, 100)))
        want = bool(_bytes(pair[0]) & _bytes(pair[1]))
        assert (mod.meets(1, *pair) == 0) == want, [(x.shape, x.stride(), x.storage_offset(), x.dtype) for x in pair]
        found[want] += 1
    assert min(found) > 500


def test_views_of_a_fused_projection():
    b, s, h, hk, d = 3, 40, 8, 2, 64
    rows = torch.zeros(b, s, h + 2 * hk, d, dtype=torch.bfloat16).permute(0, 2, 1, 3)
    heads = torch.zeros(b, h + 2 * hk, s, d, dtype=torch.bfloat16)
    for x in (rows, heads, rows[:1], rows[:, :, :1], heads[:1]):
        q, k, v = x[:, :h], x[:, h:h + hk], x[:, h + hk:]
        mod = plans.native()
        assert mod.meets(3, q, k, k, v, q, v) == -1
        assert mod.meets(9, q, k, q, x[:, h - 1:h + 1], q, q) == 1 and mod.meets(9, q, q) == 0
        assert mod.meets(0, q, q, k, k) == -1 and mod.meets(1, q, v, q, q, q, x[:, :1]) == 2
        assert mod.meets(0, q, q.view(q.shape), q, x[:, 1:h + 1]) == 1
    halves = torch.zeros(4, 9, 128)
    assert plans.native().meets(1, halves[..., :64], halves[..., 64:]) == -1
    assert plans.native().meets(1, halves[..., :64], halves[..., 60:68]) == 0


def test_what_is_no_memory_meets_nothing():
    t = torch.zeros(8)
    assert plans.native().meets(2, None, t, t, None) == -1 and plans.native().meets(2, "t", t, t[:0], t) == -1
    assert plans.native().meets(5) == -1 and plans.native().meets(1, t, torch.zeros(8, device="meta")) == -1
    with pytest.raises(TypeError):
        plans.native().meets("x", t, t)
    handwritten.apart("f", ("a", "b"), 1, t[:4], t[4:])


def _rope(h=4, hk=4):
    x = torch.zeros(2, h + hk, 8, 64, dtype=torch.bfloat16)
    w, table = torch.ones(64), torch.zeros(16, 32)
    return dict(q=x[:, :h], k=x[:, h:], q_weight=w, k_weight=w.clone(), cos=table, sin=table.clone())


def test_norm_rope_refuses_shared_outputs():
    """On CPU tensors, which would be refused next for being none of the GPU's."""
    plans.native()
    a = _rope()
    q, k, other = a["q"], a["k"], torch.zeros(2, 5, 8, 64, dtype=torch.bfloat16)
    for outs, names in (((k, q), "q_out and k have"), ((other[:, 1:], other[:, :4]), "q_out and k_out have"),
                        ((other[:, :4], other.view(2, 5, 8, 64)[:, :4]), "q_out and k_out have"),
                        ((None, q), "k_out and q have"), ((k.view(k.shape), None), "q_out and k have")):
        with pytest.raises(ValueError, match=names):
            api.qk_norm_rope(**a, q_out=outs[0], k_out=outs[1])
    with pytest.raises(ValueError, match="q_out and q have"):
        api.qk_norm_rope(**{**a, "q": other[:, 1:]}, q_out=other[:, :4])
    for outs in ((q, k), (q, None), (None, k), (other[:, :4], None), (q.view(q.shape), k)):
        with pytest.raises(ValueError, match="must be a GPU tensor"):
            api.qk_norm_rope(**a, q_out=outs[0], k_out=outs[1])


def test_norm_rope_backward_refuses_shared_outputs():
    plans.native()
    a, g = _rope(), torch.zeros(2, 9, 8, 64, dtype=torch.bfloat16)
    gq, gk = g[:, :4], g[:, 4:8]
    for given, names in ((dict(dq=gk), "dq and dk_out have"), (dict(dk=gq), "dk and dq_out have"), (dict(dq=a["k"]), "dq and k have"),
                         (dict(dk=a["q"]), "dk and q have"), (dict(dq=g[:, 1:5]), "dq and dk_out have"),
                         (dict(dk=g[:, 5:]), "dk and dk_out have"), (dict(dq=gq, dk=gq.view(gq.shape)), "dq and dk have")):
        with pytest.raises(ValueError, match=names):
            api.qk_norm_rope_backward(gq, gk, **a, **given)
    w = torch.zeros(100)
    with pytest.raises(ValueError, match="dq_weight and dk_weight have"):
        api.qk_norm_rope_backward(gq, gk, **a, dq_weight=w[:64], dk_weight=w[36:])
    for given in (dict(dq=gq, dk=gk), dict(dq=a["q"], dk=a["k"]), dict(dq=gq, dk=a["k"])):
        with pytest.raises(ValueError, match="must be a GPU tensor"):
            api.qk_norm_rope_backward(gq, gk, **a, **given)


def test_cache_calls_refuse_shared_outputs():
    plans.native()
    cache = api.KVCache.empty(4, 2, 16, 64, device="cpu")
    table, lengths = torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    x = torch.zeros(3, 5, 8, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="k and v have"):
        api.kv_cache_read(cache, table, lengths, 8, k=x[:, :2], v=x[:, 1:3])
    with pytest.raises(ValueError, match="must be a GPU tensor"):
        api.kv_cache_read(cache, table, lengths, 8, k=x[:, :2], v=x[:, 2:4])
    with pytest.raises(ValueError, match="out and q have"):
        api.attention_cached(x[:, :4], cache, table, lengths, out=x[:, 1:])
    with pytest.raises(ValueError, match="out and lse have"):
        api.attention_cached(x[:, :4].clone(), cache, table, lengths, out=x[:, :4], lse=x.view(torch.float32)[:, :4, :, 0])
    with pytest.raises(ValueError, match="must be a GPU tensor"):
        api.attention_cached(x[:, :4], cache, table, lengths, out=x[:, :4])
    with pytest.raises(ValueError, match="k_scale and cache.v_scale are one tensor"):
        api.kv_cache_write(cache._replace(v_scale=cache.k_scale), x[:, :2], x[:, 2:4], table, lengths)
