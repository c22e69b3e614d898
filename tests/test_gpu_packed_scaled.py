"""Results follow a power of two in v bit for bit, as long as sums over the keys,
which are divided at the end, fit 32 bits: probabilities over a kept maximum are up to 2^16."""
import pytest
import torch

from oracle.torch_ref import seeded_normal
from tests import test_gpu_attention_packed as attention
from tests.conftest import announce
from tests.test_gpu_packed_forms import FORMS, take   # noqa: F401 (a fixture)
from warpir_amd import api

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d,form", [(64, f) for f in FORMS[:2]] + [(128, f) for f in FORMS])
def test_large_values(gpu, take, d, form, causal):   # noqa: F811
    announce(f"packed attention D{d} {form} causal={causal}, values up to 2^96")
    take(form)
    ends = [0, 700, 730]
    q, k, v = (x.clone() for x in attention._inputs(4, 2, d, ends[-1], False))
    q[:, :, 0] = 4.0
    k[:, :700, 0] = torch.arange(700, device="cuda").bfloat16() * (0.02 * d ** 0.5)   # scores that rise from tile to tile
    v = v.clamp(-8.0, 8.0)
    offsets = torch.tensor(ends, dtype=torch.int32, device="cuda")
    o, lse = api.attention_packed(q, k, v, offsets, causal=causal)
    far, same = api.attention_packed(q, k, v * 2.0 ** 93, offsets, causal=causal)
    assert bool(far.isfinite().all()) and torch.equal(far, o * 2.0 ** 93) and torch.equal(same, lse)
