"""What the packed attention, rotation and 8-bit integer calls refuse, on the
CPU: before any launch, with the argument's name."""
import warnings

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from warpir_amd import api, handwritten, int8, packed, rotary

pytestmark = pytest.mark.filterwarnings("ignore:Accessing the data pointer of FakeTensor")

MODULES = (packed, rotary, int8)
f32, i32, i8, bf16 = torch.float32, torch.int32, torch.int8, torch.bfloat16


class _NoPlans(handwritten.DevicePlans):
    def run(self, flags, *tensors):
        return None


@pytest.fixture(autouse=True)
def never_launched(monkeypatch):
    def launch(*a, **k):
        raise AssertionError("a launch was reached")

    for module in MODULES:
        monkeypatch.setattr(module, "launch", launch)
        for name in vars(module).copy():
            if name.endswith("_plans"):
                monkeypatch.setattr(module, name, _NoPlans("none"))


@pytest.fixture
def lenient(monkeypatch):
    """The checks without the last one, which every fake tensor fails."""
    real = handwritten.check_tensor

    def check(fn, name, t, *a, **k):
        try:
            real(fn, name, t, *a, **k)
        except ValueError as e:
            if "no memory" not in str(e):
                raise
    for module in MODULES:
        monkeypatch.setattr(module, "check_tensor", check)


def _fake(*shape, dtype=bf16):
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        with FakeTensorMode():
            return torch.empty(*shape, dtype=dtype, device="cuda")


def _attend(**change):
    a = dict(q=_fake(4, 30, 64), k=_fake(2, 30, 64), v=_fake(2, 30, 64), offsets=_fake(3, dtype=i32))
    a.update(change)
    return a


@pytest.mark.parametrize("change,error", [
    (dict(q=_fake(4, 30, 96), k=_fake(2, 30, 96), v=_fake(2, 30, 96)), "64 or 128"),
    (dict(q=_fake(1, 4, 30, 64)), "q must have shape"),
    (dict(q=_fake(4, 30, 64, dtype=torch.float16)), "q must be bfloat16"),
    (dict(q=torch.zeros(4, 30, 64, dtype=bf16)), "q must be a GPU tensor"),
    (dict(q=None), "q must be a torch.Tensor"),
    (dict(k=_fake(2, 31, 64)), "k must have shape"),
    (dict(v=_fake(4, 30, 64)), "v must have shape"),
    (dict(k=_fake(3, 30, 64), v=_fake(3, 30, 64)), "not a multiple"),
    (dict(k=_fake(0, 30, 64), v=_fake(0, 30, 64)), "not a multiple"),
    (dict(q=_fake(4, 64, 30).transpose(1, 2)), "q's last dimension must be contiguous"),
    (dict(v=_fake(2, 30, 68)[..., :64]), "16-byte aligned"),
    (dict(offsets=_fake(3, dtype=torch.int64)), "offsets must be int32"),
    (dict(offsets=_fake(3, 1, dtype=i32)), "offsets must have shape"),
    (dict(offsets=_fake(0, dtype=i32)), "offsets must hold"),
    (dict(offsets=_fake(6, dtype=i32)[::2]), "offsets must be contiguous"),
    (dict(offsets=[0, 30]), "offsets must be a torch.Tensor"),
    (dict(causal=1), "causal must be a bool"),
    (dict(q=_fake(1, 1, 64).expand(1 << 12, 1 << 20, 64), k=_fake(1, 1, 64).expand(1, 1 << 20, 64),
          v=_fake(1, 1, 64).expand(1, 1 << 20, 64)), "2\\^32 threads"),
    (dict(q=_fake(1, 1, 64).expand(1, (1 << 31) - 1, 64), k=_fake(1, 1, 64).expand(1, (1 << 31) - 1, 64),
          v=_fake(1, 1, 64).expand(1, (1 << 31) - 1, 64)), "2\\^31 tokens"),
])
def test_attention(lenient, change, error):
    a = _attend(**change)
    with pytest.raises((ValueError, TypeError), match=error):
        api.attention_packed(**a)
    with pytest.raises((ValueError, TypeError), match=error):
        api.attention_packed_backward(**a, o=_fake(4, 30, 64), lse=_fake(4, 30, dtype=f32), do=_fake(4, 30, 64))


@pytest.mark.parametrize("change,error", [
    (dict(out=_fake(4, 29, 64)), "out must have shape"),
    (dict(out=_fake(4, 30, 64, dtype=f32)), "out must be bfloat16"),
    (dict(out=_fake(1, 30, 64).expand(4, 30, 64)), "out's elements overlap"),
    (dict(lse=_fake(30, 4, dtype=f32)), "lse must have shape"),
    (dict(lse=_fake(4, 1, dtype=f32).expand(4, 30)), "lse's elements overlap"),
])
def test_attention_results(lenient, change, error):
    with pytest.raises((ValueError, TypeError), match=error):
        api.attention_packed(**_attend(**change))


@pytest.mark.parametrize("change,error", [
    (dict(o=_fake(4, 31, 64)), "o must have shape"),
    (dict(do=_fake(4, 30, 64, dtype=f32)), "do must be bfloat16"),
    (dict(lse=_fake(4, 30)), "lse must be float32"),
    (dict(dq=_fake(2, 30, 64)), "dq must have shape"),
    (dict(dk=_fake(4, 30, 64)), "dk must have shape"),
    (dict(dv=_fake(2, 1, 64).expand(2, 30, 64)), "dv's elements overlap"),
    (dict(workspace=_fake(239, dtype=f32)), "workspace needs 240"),
    (dict(workspace=_fake(240)), "workspace must be float32"),
])
def test_attention_gradients(lenient, change, error):
    a = dict(o=_fake(4, 30, 64), lse=_fake(4, 30, dtype=f32), do=_fake(4, 30, 64))
    a.update(change)
    with pytest.raises((ValueError, TypeError), match=error):
        api.attention_packed_backward(**_attend(), **a)


def _axes(**change):
    a = dict(q=_fake(2, 4, 8, 64), k=_fake(2, 2, 8, 64), cos=_fake(16, 24, dtype=f32), sin=_fake(16, 24, dtype=f32),
             positions=_fake(3, 2, 8, dtype=i32), sections=(8, 8, 8))
    a.update(change)
    return a


@pytest.mark.parametrize("change,error", [
    (dict(q=_fake(2, 4, 8, 96), k=_fake(2, 2, 8, 96)), "64 or 128"),
    (dict(q=_fake(4, 8, 64)), "must have shape"),
    (dict(q=_fake(2, 4, 8, 68)[..., :64]), "16-byte aligned"),
    (dict(k=_fake(2, 2, 9, 64)), "must have shape"),
    (dict(cos=_fake(16, 32, dtype=f32)), "cos must have shape"),
    (dict(cos=_fake(0, 24, dtype=f32), sin=_fake(0, 24, dtype=f32)), "no rows"),
    (dict(sin=_fake(15, 24, dtype=f32)), "sin must have shape"),
    (dict(positions=_fake(2, 2, 8, dtype=i32)), "positions must have shape"),
    (dict(positions=_fake(3, 9, dtype=i32)), "positions must have shape"),
    (dict(positions=_fake(3, 8, dtype=torch.int16)), "positions must be int32 or int64"),
    (dict(sections=(8, 8)), "cos must have shape"),
    (dict(sections=()), "sections must be"),
    (dict(sections=24), "sections must be"),
    (dict(sections=None), "sections must be"),
    (dict(sections=(8, 8, 4, 4, 0)), "sections must be"),
    (dict(sections=(8, 24, -8)), "sections must be"),
    (dict(sections=(8.0, 8, 8)), "sections must be"),
    (dict(sections=([8], 8, 8)), "sections must be"),
    (dict(sections=(8, 8, 7)), "add up to"),
    (dict(sections=(0, 0, 0)), "add up to"),
    (dict(sections=(16, 16, 16), cos=_fake(16, 48, dtype=f32), sin=_fake(16, 48, dtype=f32)), "48 pairs do not fit"),
    (dict(interleaved=1), "interleaved must be a bool"),
    (dict(interleaved=None), "interleaved must be a bool"),
])
def test_axes(lenient, change, error):
    a = _axes(**change)
    with pytest.raises((ValueError, TypeError), match=error):
        api.rope_axes(**a)
    with pytest.raises((ValueError, TypeError), match=error):
        api.rope_axes_backward(a.pop("q"), a.pop("k"), **a)


def test_axes_results(lenient):
    one = _fake(2, 2, 8, 64)
    with pytest.raises(ValueError, match="q_out and k_out are one tensor"):
        api.rope_axes(**_axes(q=_fake(2, 2, 8, 64)), q_out=one, k_out=one)
    with pytest.raises(ValueError, match="q_out must have shape"):
        api.rope_axes(**_axes(), q_out=_fake(2, 4, 7, 64))
    with pytest.raises(ValueError, match="k_out's elements overlap"):
        api.rope_axes(**_axes(), k_out=_fake(1, 2, 8, 64).expand(2, 2, 8, 64))
    wide = [_fake(1, 1, 1, 64).expand(1 << 20, n, 1, 64) for n in (1 << 9, 1)]
    with pytest.raises(ValueError, match="2\\^29 rows"):
        api.rope_axes(**_axes(q=wide[0], k=wide[1], positions=_fake(3, 1, dtype=i32)))


@pytest.mark.parametrize("change,error", [
    (dict(x=_fake(4, 4, 32)), "x must have shape"),
    (dict(x=_fake(4, 32, dtype=f32)), "x must be bfloat16"),
    (dict(x=_fake(4, 24)), "multiple of 16"),
    (dict(x=_fake(4, 0)), "multiple of 16"),
    (dict(x=_fake(1, 131072)), "multiple of 16 up to"),
    (dict(x=_fake(32, 4).t()), "last dimension"),
    (dict(codes=_fake(4, 16, dtype=i8)), "codes must have shape"),
    (dict(codes=_fake(4, 32, dtype=torch.uint8)), "codes must be int8"),
    (dict(codes=_fake(1, 32, dtype=i8).expand(4, 32)), "codes's elements overlap"),
    (dict(codes=_fake(4, 40, dtype=i8)[:, :32]), "16-byte aligned"),
    (dict(scale=_fake(3, dtype=f32)), "scale must have shape"),
    (dict(scale=_fake(8, dtype=f32)[::2]), "scale must be contiguous"),
])
def test_quantize(lenient, change, error):
    a = dict(x=_fake(4, 32))
    a.update(change)
    with pytest.raises((ValueError, TypeError), match=error):
        api.quantize_int8(**a)


@pytest.mark.parametrize("change,error", [
    (dict(a=_fake(4, 32)), "a must be int8"),
    (dict(b=_fake(8, 48, dtype=i8)), "b must have shape"),
    (dict(a=_fake(4, 24, dtype=i8), b=_fake(8, 24, dtype=i8)), "16-byte aligned"),
    (dict(a=_fake(4, 32, dtype=i8)[:, :24], b=_fake(8, 32, dtype=i8)[:, :24]), "multiple of 16"),
    (dict(a=_fake(4, 131072, dtype=i8), b=_fake(8, 131072, dtype=i8)), "multiple of 16 up to"),
    (dict(a=_fake(4, 40, dtype=i8)[:, :32]), "16-byte aligned"),
    (dict(a_scale=_fake(8, dtype=f32)), "a_scale must have shape"),
    (dict(b_scale=_fake(8)), "b_scale must be float32"),
    (dict(b_scale=_fake(16, dtype=f32)[::2]), "b_scale must be contiguous"),
    (dict(out=_fake(4, 8, dtype=f32)), "out must be bfloat16"),
    (dict(out=_fake(8, 4).t()), "out's last dimension"),
    (dict(out=_fake(1, 8).expand(4, 8)), "out's elements overlap"),
    (dict(a=_fake(4, 1 << 23, dtype=i8)[:, :32]), "2\\^23 bytes"),
])
def test_gemm(lenient, change, error):
    a = dict(a=_fake(4, 32, dtype=i8), b=_fake(8, 32, dtype=i8), a_scale=_fake(4, dtype=f32), b_scale=_fake(8, dtype=f32))
    a.update(change)
    with pytest.raises((ValueError, TypeError), match=error):
        api.gemm_int8(**a)


def test_tensors_without_memory():
    for call, a in ((api.attention_packed, _attend()), (api.rope_axes, _axes()), (api.quantize_int8, dict(x=_fake(4, 32))),
                    (api.gemm_int8, dict(a=_fake(4, 32, dtype=i8), b=_fake(8, 32, dtype=i8), a_scale=_fake(4, dtype=f32),
                                         b_scale=_fake(8, dtype=f32)))):
        with pytest.raises(ValueError, match="no memory"):
            call(**a)
