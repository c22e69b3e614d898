"""Batches whose programs come in another order than their blocks (sequences
about as long as a block, 64 block numbers and more), and offsets that are no
offsets, with memory on all sides of what is written that has to stay.  The
checks and tolerances are those of test_gpu_attention_packed.py."""
import pytest
import torch

from oracle.torch_ref import seeded_normal
from tests import test_gpu_attention_packed as attention
from tests.conftest import announce
from tests.test_gpu_packed_forms import take   # noqa: F401 (a fixture)
from warpir_amd import api

pytestmark = pytest.mark.gpu

ORDERED = [   # form, D, query and key/value heads, rows of a workgroup of the forward
    ("split", 64, 2, 1, 32), ("split", 128, 2, 1, 32), ("four waves", 64, 3, 1, 128), ("four waves", 128, 2, 2, 128),
    ("eight waves", 128, 4, 2, 128), ("eight waves", 128, 1, 1, 256)]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("batch", [70, 131])
@pytest.mark.parametrize("form,d,h,hk,rows", ORDERED)
def test_sequences_as_long_as_a_block(gpu, take, form, d, h, hk, rows, batch, causal):   # noqa: F811
    announce(f"packed attention H{h}/{hk} D{d} {form} causal={causal}, {batch} sequences of about {rows}")
    take(form)
    gen = torch.Generator().manual_seed(batch + rows)
    lengths = torch.randint(rows // 2, 3 * rows // 2, (batch,), generator=gen).tolist()
    lengths[batch // 3], lengths[batch // 2] = 0, rows
    ends = attention._ends(lengths)
    tokens = ends[-1] + 40
    blocks = tokens // rows + batch + 1
    assert 3 * rows * batch < 4 * tokens and 2 * tokens < 3 * rows * batch and blocks > 64 and blocks % 64
    q, k, v = attention._inputs(h, hk, d, tokens, True)
    do = seeded_normal((tokens, h, d), 9).cuda().transpose(0, 1)
    offsets = torch.tensor(ends, dtype=torch.int32, device="cuda")
    o, lse = api.attention_packed(q, k, v, offsets, causal=causal)
    grads = api.attention_packed_backward(q, k, v, o, lse, do, offsets, causal=causal)
    assert bool((o[:, ends[-1]:] == 0).all()) and bool((lse[:, ends[-1]:] == -float("inf")).all())
    assert all(bool((g[:, ends[-1]:] == 0).all()) for g in grads)
    attention._check_forward(o, lse, q, k, v, ends, causal)
    attention._check_backward(grads, q, k, v, o, lse, do, ends, causal)


MARGIN = 512   # tokens


def _inside(heads, tokens, d, by_token, dtype=torch.bfloat16):
    """(all of it, the [heads, tokens, d] in the middle)"""
    n = tokens + 2 * MARGIN
    big = (torch.full((n, heads, d), 5.0, dtype=dtype, device="cuda").transpose(0, 1) if by_token
           else torch.full((heads, n, d), 5.0, dtype=dtype, device="cuda"))
    return big, big[:, MARGIN:MARGIN + tokens]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("wild", [100, 1 << 30])
@pytest.mark.parametrize("batch", [3, 70, 600])
@pytest.mark.parametrize("form,d,h,hk", [(f, d, h, hk) for f, d, h, hk, _ in ORDERED])
def test_wild_offsets_leave_what_is_around(gpu, take, form, d, h, hk, batch, wild, causal):   # noqa: F811
    announce(f"packed attention H{h}/{hk} D{d} {form} causal={causal}, {batch} offsets up to {wild} outside")
    take(form)
    t = 900
    gen = torch.Generator().manual_seed(batch)
    offsets = torch.randint(-wild, t + wild, (batch + 1,), generator=gen)
    some = torch.rand(batch + 1, generator=gen) < 0.5
    offsets = torch.where(some, torch.randint(0, t + 1, (batch + 1,), generator=gen), offsets).int().cuda()
    q, k, v = attention._inputs(h, hk, d, t, True)
    do = seeded_normal((h, t, d), 3).cuda()
    for by_token in (True, False):
        all_o, o = _inside(h, t, d, by_token)
        all_lse, lse = _inside(h, t, 1, by_token, torch.float32)
        api.attention_packed(q, k, v, offsets, causal=causal, out=o, lse=lse[..., 0])
        grads = [_inside(n, t, d, by_token) for n in (h, hk, hk)]
        ws = torch.full((2 * h * t + 2 * MARGIN * d,), 5.0, device="cuda")
        api.attention_packed_backward(q, k, v, o.nan_to_num(0.0), lse[..., 0].clamp(-50, 50), do, offsets, causal=causal,
                                      dq=grads[0][1], dk=grads[1][1], dv=grads[2][1], workspace=ws[MARGIN * d:-MARGIN * d])
        for x in (all_o, all_lse, *(g[0] for g in grads)):
            assert bool((x[:, :MARGIN] == 5.0).all()) and bool((x[:, MARGIN + t:] == 5.0).all())
        assert bool((ws[:MARGIN * d] == 5.0).all()) and bool((ws[-MARGIN * d:] == 5.0).all())
