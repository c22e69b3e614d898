"""What the layer and cache calls refuse, on the CPU: before any launch, with
the argument's name."""
import math
import warnings

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from warpir_amd import api, handwritten, kvcache, rotary

pytestmark = pytest.mark.filterwarnings("ignore:Accessing the data pointer of FakeTensor")


class _NoPlans(handwritten.DevicePlans):
    def run(self, flags, *tensors):
        return None


@pytest.fixture(autouse=True)
def never_launched(monkeypatch):
    def launch(*a, **k):
        raise AssertionError("a launch was reached")

    for module in (rotary, kvcache):
        monkeypatch.setattr(module, "launch", launch)
        for name in vars(module).copy():
            if name.endswith("_plans"):
                monkeypatch.setattr(module, name, _NoPlans("none"))


def _fake(*shape, dtype=torch.bfloat16):
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        with FakeTensorMode():
            return torch.empty(*shape, dtype=dtype, device="cuda")


f32, i32 = torch.float32, torch.int32


def _rope(**change):
    a = dict(q=_fake(2, 4, 8, 64), k=_fake(2, 2, 8, 64), q_weight=_fake(64), k_weight=_fake(64),
             cos=_fake(16, 32, dtype=f32), sin=_fake(16, 32, dtype=f32))
    a.update(change)
    return a


@pytest.mark.parametrize("change,error", [
    (dict(q=_fake(2, 4, 8, 96), k=_fake(2, 2, 8, 96)), "64 or 128"),
    (dict(q=_fake(4, 8, 64)), "q must have shape"),
    (dict(q=_fake(2, 4, 8, 64, dtype=torch.float16)), "q must be bfloat16"),
    (dict(q=torch.zeros(2, 4, 8, 64, dtype=torch.bfloat16)), "q must be a GPU tensor"),
    (dict(q="q"), "q must be a torch.Tensor"),
    (dict(k=_fake(2, 2, 9, 64)), "k must have shape"),
    (dict(q=_fake(2, 4, 64, 8).transpose(2, 3)), "q's last dimension must be contiguous"),
    (dict(q=_fake(2, 4, 8, 68)[..., :64]), "16-byte aligned"),
    (dict(q_weight=_fake(32)), "q_weight must have shape"),
    (dict(k_weight=_fake(64, dtype=f32)), "k_weight must be bfloat16"),
    (dict(cos=_fake(16, 64, dtype=f32)), "cos must have shape"),
    (dict(cos=_fake(0, 32, dtype=f32), sin=_fake(0, 32, dtype=f32)), "no rows"),
    (dict(sin=_fake(15, 32, dtype=f32)), "sin must have shape"),
    (dict(positions=_fake(2, 7, dtype=i32)), "positions must have shape"),
    (dict(positions=_fake(2, 8, dtype=torch.int16)), "positions must be int32 or int64"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps="x"), "eps"),
    (dict(interleaved=1), "interleaved"),
])
def test_norm_rope(monkeypatch, change, error):
    _lenient(monkeypatch)
    with pytest.raises((ValueError, TypeError), match=error):
        api.qk_norm_rope(**_rope(**change))
    g = dict(dq_out=_fake(2, 4, 8, 64), dk_out=_fake(2, 2, 8, 64))
    with pytest.raises((ValueError, TypeError), match=error):
        api.qk_norm_rope_backward(**g, **_rope(**change))


def _lenient(monkeypatch):
    """The checks without the last one, which every fake tensor fails."""
    real = handwritten.check_tensor

    def check(fn, name, t, *a, **k):
        try:
            real(fn, name, t, *a, **k)
        except ValueError as e:
            if "no memory" not in str(e):
                raise
    for module in (rotary, kvcache):
        monkeypatch.setattr(module, "check_tensor", check)


@pytest.mark.parametrize("change,error", [
    (dict(q_out=_fake(2, 4, 7, 64)), "q_out must have shape"),
    (dict(q_out=_fake(2, 4, 8, 64), k_out=_fake(1, 2, 8, 64).expand(2, 2, 8, 64)), "overlap"),
    (dict(positions=_fake(7, dtype=i32)), "positions must have shape"),
    (dict(q=_fake(1, 1, 1, 64).expand(1 << 20, 1 << 9, 1, 64), k=_fake(1, 1, 1, 64).expand(1 << 20, 1, 1, 64)), "2\\^29 rows"),
    (dict(q=_fake(1, 1, 1, 64).expand(1 << 24, 1, 1, 64), k=_fake(1, 1, 1, 64).expand(1 << 24, 1, 1, 64)), "2\\^24 workgroups"),
])
def test_norm_rope_past_the_pointers(monkeypatch, change, error):
    _lenient(monkeypatch)
    with pytest.raises(ValueError, match=error):
        api.qk_norm_rope(**_rope(**change))


def test_one_tensor_for_two_results():
    one = _fake(2, 2, 8, 64)
    with pytest.raises(ValueError, match="q_out and k_out are one tensor"):
        api.qk_norm_rope(**_rope(q=_fake(2, 2, 8, 64)), q_out=one, k_out=one)
    with pytest.raises(ValueError, match="dq and dk are one tensor"):
        api.qk_norm_rope_backward(one, one, **_rope(q=_fake(2, 2, 8, 64)), dq=one, dk=one)
    w = _fake(64, dtype=f32)
    with pytest.raises(ValueError, match="dq_weight and dk_weight are one tensor"):
        api.qk_norm_rope_backward(one, one, **_rope(q=_fake(2, 2, 8, 64)), dq_weight=w, dk_weight=w)
    with pytest.raises(ValueError, match="k and v are one tensor"):
        api.kv_cache_read(None, None, None, 8, k=one, v=one)


def test_norm_rope_backward_past_the_pointers(monkeypatch):
    _lenient(monkeypatch)
    g = dict(dq_out=_fake(2, 4, 8, 64), dk_out=_fake(2, 2, 8, 64), dq=_fake(2, 4, 8, 64), dk=_fake(2, 2, 8, 64),
             dq_weight=_fake(64, dtype=f32), dk_weight=_fake(64, dtype=f32))
    for change, error in ((dict(dq_out=_fake(2, 2, 8, 64)), "dq_out must have shape"),
                          (dict(dk=_fake(2, 4, 8, 64)), "dk must have shape"),
                          (dict(dq_weight=_fake(64)), "dq_weight must be float32"),
                          (dict(workspace=_fake(64, dtype=f32)), "workspace needs"),
                          (dict(workspace=_fake(10 ** 6)), "workspace must be float32")):
        with pytest.raises((ValueError, TypeError), match=error):
            api.qk_norm_rope_backward(**{**g, **_rope(), **change})


e4 = torch.float8_e4m3fn


def _cache(pages=4, heads=2, page=16, d=64, **change):
    c = dict(k=_fake(pages, heads, page, d, dtype=e4), v=_fake(pages, heads, d, page, dtype=e4),
             k_scale=_fake(pages, heads, dtype=f32), v_scale=_fake(pages, heads, dtype=f32))
    c.update(change)
    return api.KVCache(**c)


CACHE_REFUSALS = [
    (dict(cache=(1, 2)), "cache must be a KVCache"),
    (dict(cache=_cache(page=24)), "page size"),
    (dict(cache=_cache(page=256)), "page size"),
    (dict(cache=_cache(d=256)), "head size"),
    (dict(cache=_cache(k=_fake(4, 2, 16, 64, dtype=torch.uint8))), "cache.k must be float8_e4m3fn"),
    (dict(cache=_cache(v=_fake(4, 2, 16, 64, dtype=e4))), "cache.v must have shape"),
    (dict(cache=_cache(k=_fake(4, 16, 2, 64, dtype=e4).transpose(1, 2))), "cache.k must be contiguous"),
    (dict(cache=_cache(k_scale=_fake(4, 1, dtype=f32))), "cache.k_scale must have shape"),
    (dict(cache=_cache(v_scale=_fake(4, 2))), "cache.v_scale must be float32"),
    (dict(cache=_cache(pages=0)), "no pages"),
    (dict(page_table=_fake(3, dtype=i32)), "page_table must have shape"),
    (dict(page_table=_fake(3, 4, dtype=torch.int64)), "page_table must be int32"),
    (dict(page_table=_fake(4, 3, dtype=i32).t()), "page_table's last dimension"),
    (dict(lengths=_fake(2, dtype=i32)), "lengths must have shape"),
    (dict(lengths=_fake(6, dtype=i32)[::2]), "lengths must be contiguous"),
    (dict(page_table=_fake(3, 1 << 27, dtype=i32)), "2\\^30 tokens"),
]


@pytest.mark.parametrize("change,error", CACHE_REFUSALS + [
    (dict(k=_fake(3, 2, 5, 128)), "k must have shape"),
    (dict(v=_fake(3, 2, 6, 64)), "v must have shape"),
    (dict(k=_fake(3, 2, 5, 64, dtype=f32)), "k must be bfloat16"),
    (dict(counts=_fake(3, dtype=torch.int64)), "counts must be int32"),
    (dict(counts=_fake(2, dtype=i32)), "counts must have shape"),
    (dict(k=_fake(3, 2, 1, 64).expand(3, 2, 1 << 25, 64), v=_fake(3, 2, 1, 64).expand(3, 2, 1 << 25, 64),
          page_table=_fake(3, 1 << 22, dtype=i32)), "2\\^24 pages"),
])
def test_cache_write(monkeypatch, change, error):
    _lenient(monkeypatch)
    a = dict(cache=_cache(), k=_fake(3, 2, 5, 64), v=_fake(3, 2, 5, 64), page_table=_fake(3, 4, dtype=i32),
             lengths=_fake(3, dtype=i32))
    with pytest.raises((ValueError, TypeError), match=error):
        api.kv_cache_write(**{**a, **change})


@pytest.mark.parametrize("change,error", CACHE_REFUSALS + [
    (dict(tokens=-1), "tokens"), (dict(tokens=2.0), "tokens"), (dict(tokens=True), "tokens"),
    (dict(k=_fake(3, 2, 8, 64)), "k must have shape"),
    (dict(k=_fake(3, 2, 9, 64), v=_fake(3, 2, 1, 64).expand(3, 2, 9, 64)), "overlap"),
])
def test_cache_read(monkeypatch, change, error):
    _lenient(monkeypatch)
    a = dict(cache=_cache(), page_table=_fake(3, 4, dtype=i32), lengths=_fake(3, dtype=i32), tokens=9)
    with pytest.raises((ValueError, TypeError), match=error):
        api.kv_cache_read(**{**a, **change})


def test_memory_is_asked_for_last():
    a = dict(page_table=_fake(3, 4, dtype=i32), lengths=_fake(3, dtype=i32))
    with pytest.raises(ValueError, match="no memory"):
        api.kv_cache_write(_cache(), _fake(3, 2, 5, 64), _fake(3, 2, 5, 64), **a)
    with pytest.raises(ValueError, match="no memory"):
        api.kv_cache_read(_cache(), tokens=9, **a)
    with pytest.raises(ValueError, match="no memory"):
        api.qk_norm_rope(**_rope())
    with pytest.raises(ValueError, match="no memory"):
        api.qk_norm_rope_backward(_fake(2, 4, 8, 64), _fake(2, 2, 8, 64), **_rope())


def test_empty_cache_and_table():
    cache = api.KVCache.empty(3, 2, 32, 128, device="cpu")
    assert cache.k.shape == (3, 2, 32, 128) and cache.v.shape == (3, 2, 128, 32) and bool((cache.k_scale == 0).all())
    for bad in ((0, 2, 32, 128), (3, 2, 48, 128), (3, 2, 32, 96)):
        with pytest.raises(ValueError):
            api.KVCache.empty(*bad, device="cpu")
    cos, sin = api.rope_table(1 << 20, 64, device="cpu")
    assert cos.shape == (1 << 20, 32) and abs(float(cos[999999, 0]) - math.cos(999999)) < 2 ** -24
    with pytest.raises(ValueError):
        api.rope_table(0, 64, device="cpu")


@pytest.mark.parametrize("change,error", CACHE_REFUSALS + [
    (dict(q=_fake(3, 4, 5, 128)), "q must have shape"),
    (dict(q=_fake(2, 4, 5, 64)), "q must have shape"),
    (dict(q=_fake(3, 4, 5, 64, dtype=f32)), "q must be bfloat16"),
    (dict(q=_fake(3, 4, 64, 5).transpose(2, 3)), "last dimension"),
    (dict(q=_fake(3, 3, 5, 64)), "not a multiple of 2"),
    (dict(q=_fake(3, 0, 5, 64)), "not a multiple of 2"),
    (dict(counts=_fake(3, dtype=torch.int64)), "counts must be int32"),
    (dict(out=_fake(3, 4, 4, 64)), "out must have shape"),
    (dict(out=_fake(3, 1, 5, 64).expand(3, 4, 5, 64)), "overlap"),
    (dict(lse=_fake(3, 4, 5)), "lse must be float32"),
    (dict(lse=_fake(3, 4, 1, dtype=f32).expand(3, 4, 5)), "overlap"),
    (dict(page_table=_fake(3, 1 << 10, dtype=i32), workspace=_fake(64, dtype=f32)), "workspace needs"),
    (dict(page_table=_fake(3, 1 << 10, dtype=i32), workspace=_fake(1 << 24)), "workspace must be float32"),
    (dict(q=_fake(3, 4, 1, 64).expand(3, 4, 1 << 23, 64), out=_fake(3, 4, 1 << 23, 64),
          lse=_fake(3, 4, 1 << 23, dtype=f32)), "2\\^24 query rows"),
    (dict(q=_fake(3, 4, 1, 64).expand(3, 4, 1 << 20, 64), out=_fake(3, 4, 1 << 20, 64), lse=_fake(3, 4, 1 << 20, dtype=f32),
          page_table=_fake(3, 1 << 21, dtype=i32)), "2\\^30 tiles"),
    (dict(q=_fake(1, 2, 1, 64).expand(1 << 22, 2, 1, 64), out=_fake(1 << 22, 2, 1, 64), lse=_fake(1 << 22, 2, 1, dtype=f32),
          page_table=_fake(1 << 22, 1000, dtype=i32), lengths=_fake(1 << 22, dtype=i32)), "2\\^32 threads"),
])
def test_attention_cached(monkeypatch, change, error):
    _lenient(monkeypatch)
    a = dict(q=_fake(3, 4, 5, 64), cache=_cache(), page_table=_fake(3, 4, dtype=i32), lengths=_fake(3, dtype=i32),
             out=_fake(3, 4, 5, 64), lse=_fake(3, 4, 5, dtype=f32))
    with pytest.raises((ValueError, TypeError), match=error):
        api.attention_cached(**{**a, **change})


def test_attention_cached_asks_for_memory_last():
    with pytest.raises(ValueError, match="no memory"):
        api.attention_cached(_fake(3, 4, 5, 64), _cache(), _fake(3, 4, dtype=i32), _fake(3, dtype=i32))


def test_attention_forms_hold_their_bounds():
    """The kernels' launch: a known kernel, at least one program a head, and slots for what `extra` allows."""
    for rows in (1, 16, 17, 32, 33, 1000):
        for heads in (1, 7, 100, 300, 600, 5000):
            for columns, page in ((1, 16), (8, 64), (40, 128), (4096, 64)):
                for d in (64, 128):
                    block, waves, extra, least = kvcache._attention_form(rows, heads, columns, page, d)
                    assert block in (16, 32, 128) and (rows <= block or rows > 32)
                    assert waves == 4 or block == 16 or (block, d) == (32, 64) or (block, waves) in ((32, 2), (128, 8))
                    assert extra >= 0 and (least > 0) == (extra > 0)
