"""What ``attention_cached`` launches, on the CPU: calls of any size that the
kernels can take are launched, within the bounds of a launch."""
import os
import re
import warnings

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from warpir_amd import api, handwritten, kvcache
from warpir_amd.runtime import PKG_DIR

pytestmark = pytest.mark.filterwarnings("ignore:Accessing the data pointer of FakeTensor")
f32, i32, e4 = torch.float32, torch.int32, torch.float8_e4m3fn


class _NoPlans(handwritten.DevicePlans):
    def run(self, flags, *tensors):
        return None


def _fake(*shape, dtype=torch.bfloat16):
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        with FakeTensorMode():
            return torch.empty(*shape, dtype=dtype, device="cuda")


@pytest.fixture
def launches(monkeypatch):
    """The launches of a call on fake tensors: (kernel, workgroups, threads of one, arguments)."""
    seen = []
    real = handwritten.check_tensor

    def check(*a, **k):
        try:
            real(*a, **k)
        except ValueError as e:
            if "no memory" not in str(e):
                raise

    def launch(rec, device, filename, symbol, grid, block, args, tensors, offsets=None):
        assert grid[1:] == block[1:] == (1, 1)
        seen.append((symbol, grid[0], block[0], args))

    monkeypatch.setattr(kvcache, "check_tensor", check)
    monkeypatch.setattr(kvcache, "launch", launch)
    monkeypatch.setattr(kvcache, "_attention_plans", _NoPlans("none"))
    return seen


def _call(b, h, hk, t, columns, page, d):
    q, table = _fake(b, h, t, d), _fake(b, columns, dtype=i32)
    cache = api.KVCache(_fake(8, hk, page, d, dtype=e4), _fake(8, hk, d, page, dtype=e4), _fake(8, hk, dtype=f32),
                        _fake(8, hk, dtype=f32))
    workspace = _fake(max(1, api.attention_cached_workspace(q, cache, table)), dtype=f32)
    api.attention_cached(q, cache, table, _fake(b, dtype=i32), out=_fake(b, h, t, d), lse=_fake(b, h, t, dtype=f32),
                         workspace=workspace)


@pytest.mark.parametrize("b,h,hk,t,columns,page,d", [
    (32, 64, 8, 8192, 128, 64, 128),     # 2^24 query rows
    (8, 64, 8, 32768, 512, 64, 128),
    (128, 128, 16, 1024, 16, 64, 128),   # divided, a row a wave in the join
    (64, 64, 8, 4096, 64, 64, 64),
    (200, 64, 8, 20000, 400, 64, 128),
    (20000, 128, 8, 16, 40, 64, 128),    # 2^25 rows in blocks of 128
    (8192, 64, 8, 1, 16384, 64, 128),    # 2^30 tiles in a table for a million tokens
    (65536, 32, 8, 1, 400, 64, 64),      # half a million heads of one block
    (4096, 64, 1, 64, 80, 64, 128),
])
def test_large_calls_are_launched(launches, b, h, hk, t, columns, page, d):
    _call(b, h, hk, t, columns, page, d)
    symbol, grid, threads, args = launches[0]
    items = b * hk * args.blocks
    assert grid == items + args.extra and grid * threads < 1 << 32
    assert len(launches) == (2 if args.extra else 1)
    for symbol, grid, threads, args in launches[1:]:
        assert grid * threads < 1 << 32 and items * -(-columns * page // 64) < 1 << 30


def test_what_cannot_be_divided_is_not():
    """The sums of a division and the grid of its join have to hold for every form."""
    for rows in (1, 8, 16, 32, 64, 1000, 100000):
        for heads in (1, 100, 1 << 16, 1 << 20, 1 << 23):
            for columns, page in ((4, 16), (400, 64), (16384, 64), (1 << 21, 128)):
                for d in (64, 128):
                    block, waves, extra, least = kvcache._attention_form(rows, heads, columns, page, d)
                    items = heads * -(-rows // block)
                    if extra:
                        assert items * -(-columns * page // 64) < 1 << 30
                        assert kvcache._join_grid(items, rows, block)[0] < 1 << 24 and least > 0
                    assert (block, waves) == kvcache._fastest_form(rows, heads, columns, page, d)[:2]


@pytest.mark.parametrize("b,h,hk,t,columns,d", [
    (64, 32, 8, 300, 7, 128), (64, 64, 4, 300, 7, 64), (500, 64, 4, 64, 2, 128), (500, 64, 4, 40, 10, 128),
    (100, 128, 16, 1000, 16, 128), (256, 128, 8, 272, 6, 64), (200, 32, 8, 64, 4, 128), (500, 16, 16, 64, 2, 64)])
def test_blocks_that_fill_the_chip_are_not_divided(b, h, hk, t, columns, d):
    """Every program of a division adds up all blocks' tiles: 2 to 6 times these launches' time, undivided."""
    block, waves, extra, least = kvcache._attention_form(t * h // hk, b * hk, columns, 64, d)
    assert b * hk * -(-t * h // hk // block) > 512 and extra == 0


@pytest.mark.parametrize("b,h,hk,t,d", [(1024, 32, 8, 1, 128), (96, 32, 8, 1, 128), (512, 32, 8, 8, 128),
                                        (512, 16, 16, 1, 64), (100, 32, 8, 8, 64), (40, 32, 32, 1, 128)])
def test_heads_that_fill_the_chip_are_not_divided_for_the_width_of_the_table(b, h, hk, t, d):
    """Short sequences in a table for long ones: a division took up to ten times the time of the narrow table's form."""
    for columns in (1, 16, 512, 16384):
        assert kvcache._attention_form(t * h // hk, b * hk, columns, 64, d)[2] == 0


def test_every_form_has_its_kernels_and_its_workspace():
    """Names that attn_cached.hip defines, with the waves and rows that it gives them; a slot for every partial result."""
    with open(os.path.join(PKG_DIR, "csrc", "attn_cached.hip")) as f:
        source = f.read()
    attention = {m[0]: [int(x) for x in m[1:6]] for m in
                 re.findall(r"^ATTN_KERNEL\((\w+), (\d+), (\d+), (\d+), (\d+), (\d+), \w+\)", source, re.M)}
    join = {m[0]: [int(x) for x in m[1:]] for m in re.findall(r"^JOIN_KERNEL\((\w+), (\d+), (\d+), (\d+)\)", source, re.M)}
    assert len(attention) > 15 and len(join) > 5
    used = set()
    for d in (64, 128):
        for rows in (1, 2, 5, 8, 16, 17, 24, 32, 33, 40, 64, 100, 128, 129, 200, 256, 400, 700, 1000, 2048, 5000, 20000):
            for heads in (1, 2, 4, 7, 8, 16, 32, 60, 100, 104, 106, 200, 256, 257, 300, 384, 385, 512, 513, 600, 768, 1100, 5000):
                for columns, page in ((1, 16), (4, 16), (2, 128), (8, 64), (20, 32), (40, 128), (300, 64), (4096, 64)):
                    block, waves, extra, least = kvcache._attention_form(rows, heads, columns, page, d)
                    items = heads * -(-rows // block)
                    grid, many = kvcache._join_grid(items, rows, block)
                    names = kvcache._attention_kernels(block, waves, extra, d, page, many)
                    used.update(names)
                    _, nq, wr, w, _ = attention[names[0]]
                    assert attention[names[0]][0] == d and (w, 16 * nq * wr) == (waves, block)
                    assert rows <= block or rows > 32   # up to 32 rows: one block
                    assert len(names) == 1 + (extra > 0) and (least > 0) == (extra > 0)
                    floats = kvcache._workspace_floats(extra, block, d, items)
                    if not extra:
                        assert floats == 0
                        continue
                    assert join[names[1]] == [d, block, 4 if many else 1]
                    assert grid * (4 if many else 1) >= items * min(rows, block)
                    # wir_pages.h: slots_for(extra) = 3 extra + 2 partial results, a row of each D values, a maximum and a sum
                    assert floats >= (3 * extra + 2) * block * (d + 2) + 4 * items
                    assert (floats - 4 * items) % 4 == 0
    assert used == set(attention) | set(join)
