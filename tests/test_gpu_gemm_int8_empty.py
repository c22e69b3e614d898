"""Sums of no products: 0, scaled as any other sum."""
import math

import pytest
import torch

from tests.conftest import announce
from warpir_amd import api

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n", [(1, 1), (3, 70), (200, 9)])
def test_no_columns(gpu, m, n):
    announce(f"gemm int8 {m} x {n} x 0")
    sa, sb = torch.ones(m, device="cuda"), torch.ones(n, device="cuda")
    a, b = (torch.empty(r, 0, dtype=torch.int8, device="cuda") for r in (m, n))
    assert bool((api.gemm_int8(a, b, sa, sb) == 0).all())
    sa[m - 1], sb[n // 2] = math.nan, math.inf
    wide = torch.full((m, n + 8), 5.0, dtype=torch.bfloat16, device="cuda")
    for out in (None, wide[:, :n]):
        got = api.gemm_int8(a, b, sa, sb, out=out)
        want = torch.zeros(m, n, device="cuda")
        want[m - 1], want[:, n // 2] = math.nan, math.nan
        assert torch.equal(got.isnan(), want.isnan()) and bool((got[~want.isnan()] == 0).all())
    assert bool((wide[:, n:] == 5.0).all())
