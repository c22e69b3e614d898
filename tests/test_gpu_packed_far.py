"""Tensors whose offsets pass 32 bits: what lies at their ends is as right (attention: against the 64-bit oracle, with the
other tests' tolerances), and has the bits (the rest), as in a tensor of its own."""
import pytest
import torch

from oracle.torch_ref import seeded_normal
from tests import test_gpu_attention_packed as attention
from tests.conftest import announce
from warpir_amd import api

pytestmark = pytest.mark.gpu

FAR = 1 << 31   # elements


@pytest.fixture(autouse=True)
def free():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("d,token_first", [(128, True), (64, False)])
def test_attention(gpu, d, token_first):
    announce(f"packed attention over 2^31 elements, D{d}")
    h, hk, n = 16, 4, 150
    t = FAR // (h * d) + 4 * n
    make = (lambda: torch.zeros(t, h, d, dtype=torch.bfloat16, device="cuda").transpose(0, 1)) if token_first else (
        lambda: torch.zeros(h, t, d, dtype=torch.bfloat16, device="cuda"))
    q, do = make(), make()
    k, v = (torch.zeros(hk, t, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    last = [seeded_normal((x.shape[0], n, d), i).cuda() for i, x in enumerate((q, k, v, do))]
    for x, y in zip((q, k, v, do), last):
        x[:, -n:] = y
    offsets = torch.cat((torch.arange(0, t - n, 512, device="cuda"), torch.tensor([t - n, t], device="cuda"))).int()
    o, lse = api.attention_packed(q, k, v, offsets)
    grads = api.attention_packed_backward(q, k, v, o, lse, do, offsets)
    attention._check_forward(o[:, -n:], lse[:, -n:], *last[:3], [0, n], True)
    attention._check_backward([x[:, -n:] for x in grads], *last[:3], o[:, -n:], lse[:, -n:], last[3], [0, n], True)
    assert bool((o[:, :1024] == 0).all()) and all(bool((x[:, :1024] == 0).all()) for x in grads)


def test_rotation(gpu):
    announce("rotation over 2^31 elements")
    h, d, n = 32, 128, 100
    t = FAR // (h * d) + n
    q = torch.zeros(1, h, t, d, dtype=torch.bfloat16, device="cuda")
    k = torch.zeros(1, t, 2, d, dtype=torch.bfloat16, device="cuda").transpose(1, 2)
    q[:, :, -n:], k[:, :, -n:] = seeded_normal((1, h, n, d), 0).cuda(), seeded_normal((1, 2, n, d), 1).cuda()
    cos, sin = api.rope_table(1000, d)
    positions = (torch.arange(t, device="cuda") % 1000).repeat(2, 1)
    want = api.rope_axes(q[:, :, -n:].contiguous(), k[:, :, -n:].contiguous(), cos, sin, positions[:, -n:].contiguous(), (24, 40))
    got = api.rope_axes(q, k, cos, sin, positions, (24, 40), q_out=q, k_out=k)
    assert got[0] is q
    assert torch.equal(q[:, :, -n:], want[0]) and torch.equal(k[:, :, -n:], want[1]) and bool((q[:, :, :-n:4096] == 0).all())


def test_codes_and_product(gpu):
    announce("quantize and gemm int8 over 2^31 elements")
    width, n = 8192, 70
    rows = FAR // width + n
    x = torch.zeros(rows, width, dtype=torch.bfloat16, device="cuda")
    x[-n:] = seeded_normal((n, width), 0).cuda()
    codes, scale = api.quantize_int8(x)
    want, want_scale = api.quantize_int8(x[-n:])
    assert torch.equal(codes[-n:], want) and torch.equal(scale[-n:], want_scale)
    del x
    b, bs = api.quantize_int8(seeded_normal((100, width), 1).cuda())
    ref = api.gemm_int8(want, b, want_scale, bs)
    out = api.gemm_int8(codes, b, scale, bs)
    assert torch.equal(out[-n:], ref) and bool((out[:1000] == 0).all())
    out = api.gemm_int8(b, codes, bs, scale)          # as a weight, and with an output past 2^31
    assert torch.equal(out[:, -n:], ref.T)
    a = torch.zeros(9000, 16, dtype=torch.int8, device="cuda")
    a[-n:] = want[:, :16]
    w = torch.zeros(FAR // 9000 + n, 16, dtype=torch.int8, device="cuda")
    w[-n:] = codes[-n:, 16:32]
    ones = torch.ones(w.shape[0], device="cuda")
    out = api.gemm_int8(a, w, ones[:9000], ones)
    assert torch.equal(out[-n:, -n:], (a[-n:].float() @ w[-n:].float().T).bfloat16())
