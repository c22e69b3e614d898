"""Keys whose scores are -inf: they weigh nothing, also where they are a row's
first ones, and a row that sees only such keys has no sum.

The oracle has -1e30 in the place of the keys' infinity, whose probabilities are 0
in 64 bits; the tolerances are those of the finite keys (test_gpu_attention_packed.py)."""
import math

import pytest
import torch

from oracle.packed_ref import packed_attention_bwd_ref, packed_attention_ref
from oracle.torch_ref import seeded_normal
from tests import test_gpu_attention_packed as attention
from tests.conftest import announce
from tests.test_gpu_packed_forms import FORMS, take   # noqa: F401 (a fixture)
from warpir_amd import api

pytestmark = pytest.mark.gpu

U = attention.U


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d,form", [(64, f) for f in FORMS[:2]] + [(128, f) for f in FORMS])
@pytest.mark.parametrize("h,hk,hidden,length", [(4, 2, 64, 100), (2, 2, 130, 333), (4, 1, 200, 230)])
def test_first_keys_weigh_nothing(gpu, take, h, hk, hidden, length, d, form, causal):   # noqa: F811
    announce(f"packed attention H{h}/{hk} D{d} {form} causal={causal}, {hidden} of {length} keys have scores of -inf")
    take(form)
    ends = [0, 40, 40 + length, 60 + length]
    q, k, v = (x.clone() for x in attention._inputs(h, hk, d, ends[-1], False))
    seq, first, tail = slice(40, 40 + length), slice(40, 40 + hidden), slice(40 + hidden, 40 + length)
    q[:, seq, 0] = q[:, seq, 0].abs() + 0.5
    k[:, first, 0] = -math.inf
    do = seeded_normal(q.shape, 9).cuda()
    offsets = torch.tensor(ends, dtype=torch.int32, device="cuda")
    o, lse = api.attention_packed(q, k, v, offsets, causal=causal)
    grads = api.attention_packed_backward(q, k, v, o, lse, do, offsets, causal=causal)

    known = k.cpu().double()
    known[:, first, 0] = -1e30
    cq, cv, cdo = (x.cpu().double() for x in (q, v, do))
    ref, ref_lse, weight, _ = packed_attention_ref(cq, known, cv, ends, causal)
    some = torch.ones(ends[-1], dtype=torch.bool)   # rows that see a key with a score
    if causal:
        some[first] = False
        assert bool((lse[:, first] == -math.inf).all()) and bool(o[:, first].isnan().all())
    known_finite = known.clone()
    known_finite[:, first] = 0
    _, _, _, scores = packed_attention_ref(cq, known_finite, cv, ends, False)
    e = 2 * (d + 8) * U * scores + 2 ** -20
    off = (o.cpu().double() - ref).abs()
    tol = 2 ** -8 * ref.abs() + (2 ** -8 + 2 * e[..., None] + 4 * length * U) * weight
    assert bool((off <= tol)[:, some].all()), off[:, some].max()
    off = (lse.cpu().double() - ref_lse).abs()
    assert bool((off <= e + 2 * length * U + 4 * U * ref_lse.abs())[:, some].all()), off[:, some].max()

    # gradients, from the outputs as they are (rows without a key with a score: any numbers, their keys are not compared)
    co, clse = o.cpu().double(), lse.cpu().double()
    co[:, ~some], clse[:, ~some] = 0.0, 0.0
    refs, bounds, noise = packed_attention_bwd_ref(cq, known, cv, co, clse, cdo, ends, causal)
    e = 2 * (d + 8) * U * float((scores + clse.abs()).max()) + 2 ** -20
    n = length * (h // hk)
    for name, got, r, bound, noisy in zip(("dq", "dk", "dv"), grads, refs, bounds, noise):
        off = (got.cpu().double() - r).abs()
        tol = 2 ** -8 * r.abs() + (2 ** -8 + 2 * e + 4 * n * U) * bound + n * 2 ** -102
        if name != "dv":
            tol += (d + 8) * U * noisy
        fine = off <= tol
        if name == "dq":   # 0 times the infinite values of column 0
            assert bool(got[:, seq, 0].isnan().all())
            fine[:, seq, 0] = True
        if causal:
            assert bool(got[:, first].isnan().all())
            fine[:, first] = True
        elif name != "dq":
            assert bool((got[:, first] == 0).all())
        assert bool(fine.all()), name
        assert bool(got[:, tail, 1:].isfinite().all())


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d,form", [(64, f) for f in FORMS[:2]] + [(128, f) for f in FORMS])
def test_no_key_has_a_score(gpu, take, d, form, causal):   # noqa: F811
    """LSE is the logarithm of 0 and O its quotient: -inf and NaN in every form; other sequences keep their bits."""
    announce(f"packed attention D{d} {form} causal={causal}, no key has a score")
    take(form)
    ends = [0, 70, 370, 400]
    q, k, v = (x.clone() for x in attention._inputs(4, 2, d, ends[-1], False))
    q[:, 70:370, 0] = q[:, 70:370, 0].abs() + 0.5
    offsets = torch.tensor(ends, dtype=torch.int32, device="cuda")
    want = api.attention_packed(q, k, v, offsets, causal=causal)
    k[:, 70:370, 0] = -math.inf
    o, lse = api.attention_packed(q, k, v, offsets, causal=causal)
    assert bool(o[:, 70:370].isnan().all()) and bool((lse[:, 70:370] == -math.inf).all())
    for at in (slice(0, 70), slice(370, 400)):
        assert torch.equal(o[:, at], want[0][:, at]) and torch.equal(lse[:, at], want[1][:, at])


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("value", [math.inf, -math.inf])
@pytest.mark.parametrize("d,form", [(64, f) for f in FORMS[:2]] + [(128, f) for f in FORMS])
def test_rows_that_see_an_infinite_key(gpu, take, d, form, value, causal):   # noqa: F811
    """Column 0 of one key is infinite: rows of the other sign there have a score of -inf and go on without it, rows of
    its sign have +inf and no results; the gradients are numbers where no such row has a part."""
    announce(f"packed attention D{d} {form} causal={causal}, a key has {value}")
    take(form)
    h, hk, ends, at = 4, 2, [0, 100, 400, 430], 177
    q, k, v = (x.clone() for x in attention._inputs(h, hk, d, ends[-1], False))
    k[:, at, 0] = value
    do = seeded_normal(q.shape, 9).cuda()
    offsets = torch.tensor(ends, dtype=torch.int32, device="cuda")
    o, lse = api.attention_packed(q, k, v, offsets, causal=causal)
    grads = api.attention_packed_backward(q, k, v, o, lse, do, offsets, causal=causal)

    tokens = torch.arange(ends[-1])
    sees = (tokens >= (at if causal else 100)) & (tokens < 400)
    cq, ck, cv = (x.cpu().double() for x in (q, k, v))
    bad = sees & (cq[:, :, 0] * value > 0)                  # [H, T]
    assert bool(o[bad].isnan().all()) and not bool(lse[bad].isfinite().any())
    # to the others the key is as far away as one can be; its scores with rows of its sign are not compared
    ck[:, at, 0] = 0
    _, _, _, scores = packed_attention_ref(cq, ck, cv, ends, False)
    ck[:, at, 0] = math.copysign(1e30, value)
    ref, ref_lse, weight, _ = packed_attention_ref(cq, ck, cv, ends, causal)
    e = 2 * (d + 8) * U * scores + 2 ** -20
    off, tol = (o.cpu().double() - ref).abs(), 2 ** -8 * ref.abs() + (2 ** -8 + 2 * e[..., None] + 4 * 300 * U) * weight
    assert bool((off <= tol)[~bad].all()), off[~bad].max()
    off = (lse.cpu().double() - ref_lse).abs()
    assert bool((off <= e + 2 * 300 * U + 4 * U * ref_lse.abs())[~bad].all()), off[~bad].max()

    dq, dk, dv = (g.cpu() for g in grads)
    assert bool(dq[bad].isnan().all()) and bool(dq[~bad][:, 1:].isfinite().all())
    assert torch.equal(dq[~bad][:, 0].isnan(), sees.expand(h, -1)[~bad])    # 0 times the infinity
    for j in range(hk):
        rows = bad[2 * j:2 * j + 2].any(0)
        hit = (tokens >= 100) & (tokens < 400) & ((tokens <= int(tokens[rows].max())) if causal else bool(rows.any()))
        assert bool(dk[j, hit].isnan().all()) and bool(dv[j, hit].isnan().all())
        assert bool(dk[j, ~hit].isfinite().all()) and bool(dv[j, ~hit].isfinite().all())
