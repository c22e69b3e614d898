"""Writing into pages whose scale is none yet, no number or no power of two:
codes of K and of V, word by word, against the 64-bit oracle.

A scale s that is kept and no power of two takes x to a code as x * (1 / s) in
fp32, off by 2^-23 of itself before the code's rounding.  So a code differs
from the oracle's only where x / s is that near a tie, and by one step.  A code
that is rounded again, c * (was / scale), likewise."""
import math

import pytest
import torch

from oracle.layer_ref import cache_write_ref
from oracle.torch_ref import seeded_normal
from tests.conftest import announce
from warpir_amd import api

pytestmark = pytest.mark.gpu
POWERS = (0.0, math.nan, 2.0 ** -140, 2.0 ** -100, 2.0 ** -9, 2.0 ** 20)
OTHERS = (1e-30, 0.3, 3e-3, 1e4)


def _pair(old, page, d, first, tokens, seed=0):
    """The cache after a write behind `first` held tokens, here and by the oracle."""
    gen = torch.Generator().manual_seed(seed)
    codes = [torch.randint(0, 256, s, generator=gen, dtype=torch.uint8) for s in ((3, 2, page, d), (3, 2, d, page))]
    codes = [torch.where(c & 127 == 127, c ^ 1, c).view(torch.float8_e4m3fn) for c in codes]
    ref = api.KVCache(*codes, *(torch.full((3, 2), old) for _ in "kv"))
    got = api.KVCache(*(x.cuda() for x in ref))
    table = torch.tensor([[2, 0]], dtype=torch.int32)
    lengths = torch.tensor([first + tokens], dtype=torch.int32)
    k, v = seeded_normal((1, 2, tokens, d), seed + 1), seeded_normal((1, 2, tokens, d), seed + 2, 5.0)
    api.kv_cache_write(got, k.cuda(), v.cuda(), table.cuda(), lengths.cuda())
    cache_write_ref(ref, k, v, table, lengths)
    return [x.cpu() for x in got], list(ref)


def _order(codes):
    """Codes as integers in the order of their values (both zeros are 0)."""
    c = codes.view(torch.uint8).int()
    return torch.where(c >= 128, 128 - c, c)


@pytest.mark.parametrize("page,d", [(16, 64), (16, 128), (32, 64), (32, 128), (64, 64), (64, 128), (128, 64), (128, 128)])
def test_codes_for_every_old_scale(gpu, page, d):
    announce(f"kv write over old scales, page {page} D{d}")
    for first, tokens in ((page // 2 + 1, 3), (1, 1), (page - 1, 5), (6, page - 7), (4, 4), (3, page)):
        for old in POWERS + OTHERS:
            got, ref = _pair(old, page, d, first, tokens)
            for name, x, y in zip(api.KVCache._fields[2:], got[2:], ref[2:]):
                assert torch.equal(x.isnan(), y.isnan()) and torch.equal(x.nan_to_num(), y.nan_to_num()), (name, old)
            for name, x, y in zip("kv", got, ref):
                assert torch.equal(x.float().isnan(), y.float().isnan()), (name, old)
                off = (_order(x) - _order(y))[~x.float().isnan()].abs()
                if old in OTHERS:
                    assert off.max() <= 1 and (off > 0).float().mean() <= 1e-3, (name, old)
                else:
                    assert off.max() == 0, (name, old)
