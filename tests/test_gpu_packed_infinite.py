"""Infinite values in the gradients: what a sum of them is by the definition, in
every form, whether or not a workgroup has to look at its values twice."""
import math

import pytest
import torch

from oracle.torch_ref import seeded_normal
from tests import test_gpu_attention_packed as attention
from tests.conftest import announce
from tests.test_gpu_packed_forms import FORMS, take   # noqa: F401 (a fixture)
from warpir_amd import api

pytestmark = pytest.mark.gpu

ENDS = [0, 100, 300, 370]


def _same(x, y):
    return torch.equal(x.nan_to_num(77.0, 88.0, 99.0), y.nan_to_num(77.0, 88.0, 99.0))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d,form", [(64, f) for f in FORMS[:2]] + [(128, f) for f in FORMS])
@pytest.mark.parametrize("at", [177, 299, 128])   # inside a block, a sequence's last token, near a block's first
def test_infinite_output_gradient(gpu, take, at, d, form, causal):   # noqa: F811
    """One infinite value of dO, row `at` of head 1, column 5.  dV of the keys that the row sees has it in that column;
    dK_j is dS_j q with dS_j = P_j (dO_5 v_j5 - dO_5 O_5): infinite where the signs of v_j5 and O_5 differ, else no number."""
    take(form)
    q, k, v = attention._inputs(4, 2, d, ENDS[-1], True)
    do = seeded_normal((4, ENDS[-1], d), 7).cuda()
    offsets = torch.tensor(ENDS, dtype=torch.int32, device="cuda")
    o, lse = api.attention_packed(q, k, v, offsets, causal=causal)
    want = api.attention_packed_backward(q, k, v, o, lse, do, offsets, causal=causal)
    tokens = torch.arange(ENDS[-1], device="cuda")
    sees = (tokens >= 100) & (tokens < 300) & (tokens <= (at if causal else 299))
    for value in (math.inf, -math.inf):
        announce(f"packed attention backward D{d} {form} causal={causal}, dO of token {at} has {value}")
        bad = do.clone()
        bad[1, at, 5] = value
        dq, dk, dv = api.attention_packed_backward(q, k, v, o, lse, bad, offsets, causal=causal)
        expected = want[2].clone()
        expected[0, sees, 5] = value
        assert torch.equal(dv, expected)
        expected = want[1].clone()
        opposite = v[0, sees, 5].sign() * o[1, at, 5].sign() < 0
        rows = torch.full((int(sees.sum()), d), math.nan, dtype=torch.bfloat16, device="cuda")
        rows[opposite] = (value * v[0, sees, 5].sign()[opposite, None] * q[1, at].sign()).bfloat16()
        expected[0, sees] = rows
        assert _same(dk, expected)
        assert bool(dq[1, at].isnan().all())
        others = dq.clone()
        others[1, at] = want[0][1, at]
        assert torch.equal(others, want[0])


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d,form", [(64, f) for f in FORMS[:2]] + [(128, f) for f in FORMS])
def test_infinite_output_gradients_of_both_signs(gpu, take, d, form, causal):   # noqa: F811
    """Keys that see +inf and -inf in a column of dO have no number there, those that see one of them have that; a NaN
    behind them reaches the keys up to it."""
    announce(f"packed attention backward D{d} {form} causal={causal}, dO has both infinities")
    take(form)
    q, k, v = attention._inputs(4, 2, d, ENDS[-1], True)
    do = seeded_normal((4, ENDS[-1], d), 7).cuda()
    offsets = torch.tensor(ENDS, dtype=torch.int32, device="cuda")
    o, lse = api.attention_packed(q, k, v, offsets, causal=causal)
    want = api.attention_packed_backward(q, k, v, o, lse, do, offsets, causal=causal)[2]
    do[0, 150, 3], do[1, 190, 3] = math.inf, -math.inf          # two heads of one key/value head
    do[2, 260, 7], do[3, 120, 7] = math.inf, math.nan
    do[2, 200, 9], do[2, 280, 9] = math.inf, math.inf
    dv = api.attention_packed_backward(q, k, v, o, lse, do, offsets, causal=causal)[2]
    expected = want.clone()
    if causal:
        expected[0, 100:191, 3], expected[0, 100:151, 3] = -math.inf, math.nan
        expected[1, 100:261, 7], expected[1, 100:121, 7] = math.inf, math.nan
        expected[1, 100:281, 9] = math.inf
    else:
        expected[0, 100:300, 3] = expected[1, 100:300, 7] = math.nan
        expected[1, 100:300, 9] = math.inf
    assert _same(dv, expected)


@pytest.mark.parametrize("d,form", [(64, f) for f in FORMS[:2]] + [(128, f) for f in FORMS])
def test_infinite_value_of_a_key_without_weight(gpu, take, d, form):   # noqa: F811
    """Row 1 of two tokens: P of key 0 is too small for 32 bits, its value infinite.  dS = P (inf - inf) is no number
    all the same, and dQ with it."""
    announce(f"packed attention backward D{d} {form}, an infinite value of a key without weight")
    take(form)
    q, k, v = (x.clone() for x in attention._inputs(2, 1, d, 2, False))
    q[:, 1, 0], k[:, 0, 0], k[:, 1, 0] = 100.0, -100.0, 1.0
    v[:, 0, 3] = math.inf
    do = seeded_normal((2, 2, d), 7).cuda()
    offsets = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    o, lse = api.attention_packed(q, k, v, offsets)
    assert bool((o[:, 1, 3] == math.inf).all())
    for causal in (True, False):
        dq = api.attention_packed_backward(q, k, v, o, lse, do, offsets, causal=causal)[0]
        assert bool(dq[:, 1].isnan().all())
