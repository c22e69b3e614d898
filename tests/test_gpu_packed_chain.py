"""The packed operators one after another, as a layer uses them: every stage
against its oracle on what the stage before it gave."""
import math

import pytest
import torch

from oracle.packed_ref import axes_angles_ref, gemm_int8_ref, rope_axes_ref
from oracle.torch_ref import seeded_normal
from tests.conftest import announce
from tests.test_gpu_attention_packed import _check_backward, _check_forward, _ends
from warpir_amd import api

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,h,hk,sections", [(64, 4, 2, (8, 8)), (128, 4, 4, (16, 24, 24))])
def test_packed_layer(gpu, d, h, hk, sections):
    """Tokens in 8 bits -> fused projection -> rotation in place -> attention -> projection, and back to the projection."""
    announce(f"packed layer H{h}/{hk} D{d} {sections}")
    ends, width = _ends([90, 1, 0, 150]), 256
    t = ends[-1]
    offsets = torch.tensor(ends, dtype=torch.int32, device="cuda")
    x = seeded_normal((t, width), 0).cuda()
    wqkv = api.quantize_int8((seeded_normal(((h + 2 * hk) * d, width), 1).float() / math.sqrt(width)).bfloat16().cuda())
    wo = api.quantize_int8((seeded_normal((width, h * d), 2).float() / math.sqrt(h * d)).bfloat16().cuda())
    codes, scale = api.quantize_int8(x)
    qkv = api.gemm_int8(codes, wqkv[0], scale, wqkv[1])
    ref = gemm_int8_ref(codes.cpu(), wqkv[0].cpu(), scale.cpu(), wqkv[1].cpu())
    assert bool(((qkv.cpu().double() - ref).abs() <= (2 ** -8 + 2 ** -21) * ref.abs()).all())

    heads = qkv.view(t, h + 2 * hk, d).transpose(0, 1)
    q, k, v = heads[:h], heads[h:h + hk], heads[h + hk:]
    before = q.clone(), k.clone()
    pos = torch.stack([(torch.arange(t, device="cuda") // (3 ** a)) % 50 for a in range(len(sections))]).int()
    freq = torch.cat([100.0 ** (-torch.arange(n, dtype=torch.float64) / n) for n in sections])
    angle = torch.arange(50, dtype=torch.float64)[:, None] * freq
    table = angle.cos().float().cuda(), angle.sin().float().cuda()
    qr, kr = api.rope_axes(q[None], k[None], *table, pos, sections, q_out=q[None], k_out=k[None])
    turned = axes_angles_ref(pos.cpu()[:, None], freq, sections)
    for got, x0 in ((qr, before[0]), (kr, before[1])):
        want, bound = rope_axes_ref(x0.cpu()[None], turned)
        assert bool(((got.cpu().double() - want).abs() <= 2 ** -8 * want.abs() + 2 ** -22 * bound).all())

    o, lse = api.attention_packed(q, k, v, offsets)
    _check_forward(o, lse, q, k, v, ends, True)
    flat = o.transpose(0, 1).reshape(t, h * d)
    assert flat.data_ptr() == o.data_ptr()      # (no copy)
    codes, scale = api.quantize_int8(flat)
    y = api.gemm_int8(codes, wo[0], scale, wo[1])
    ref = gemm_int8_ref(codes.cpu(), wo[0].cpu(), scale.cpu(), wo[1].cpu())
    assert bool(((y.cpu().double() - ref).abs() <= (2 ** -8 + 2 ** -21) * ref.abs()).all())

    do = seeded_normal((t, h, d), 9).cuda().transpose(0, 1)
    dqkv = torch.empty_like(qkv).view(t, h + 2 * hk, d).transpose(0, 1)
    dq, dk, dv = dqkv[:h], dqkv[h:h + hk], dqkv[h + hk:]
    api.attention_packed_backward(q, k, v, o, lse, do, offsets, dq=dq, dk=dk, dv=dv)
    _check_backward((dq, dk, dv), q, k, v, o, lse, do, ends, True)
    gq, gk = dq.clone(), dk.clone()
    api.rope_axes_backward(dq[None], dk[None], *table, pos, sections, dq=dq[None], dk=dk[None])
    for got, g in ((dq, gq), (dk, gk)):
        want, bound = rope_axes_ref(g.cpu()[None], turned, back=True)
        assert bool(((got.cpu().double()[None] - want).abs() <= 2 ** -8 * want.abs() + 2 ** -22 * bound).all())
    assert api.gemm(dqkv.transpose(0, 1).reshape(t, -1), torch.zeros((h + 2 * hk) * d, 64, dtype=torch.bfloat16,
                                                                     device="cuda")).shape == (t, 64)


def test_one_sequence_is_dense_attention(gpu):
    """The dense kernels' results, within the two kernels' tolerances against one another: both round the same
    probabilities to bf16 (2^-8 of sum P |v| each, and 2^-8 of the result)."""
    q, k, v = (seeded_normal((1, n, 256, 128), i).cuda() for i, n in enumerate((4, 2, 2)))
    for causal in (False, True):
        want, want_lse = api.attention_forward(q, k, v, causal=causal)
        o, lse = api.attention_packed(q[0], k[0], v[0], torch.tensor([0, 256], dtype=torch.int32, device="cuda"), causal=causal)
        bound = 2 ** -7 * want[0].float().abs() + 2 ** -6 * v.float().abs().amax()
        assert bool(((o.float() - want[0].float()).abs() <= bound).all())
        assert bool(((lse - want_lse[0]).abs() <= 1e-4).all())
