"""The rules that choose a kernel by sizes, on the CPU: each form is chosen somewhere in the calls' range, and none that is not built."""
import os

import pytest

from warpir_amd import int8, packed

SIZES = (1, 7, 16, 17, 33, 64, 65, 130, 500, 777, 1024, 2000, 4096, 10000, 16384, 40000)


def test_product_tiles():
    named = {int8._gemm_form(m, n, k) for m in SIZES for n in (1, 64, 1000, 4096, 5000, 6144, 8192, 16384, 40000)
             for k in (16, 512, 4096, 14336)}
    assert {f[0] for f in named if f[0] in int8._TILES} == set(int8._TILES)
    assert ("64_split", 64, 64, 256) in named
    assert all(f[1:] == int8._TILES[f[0]][:3] for f in named if f[0] in int8._TILES)
    few = {f[0] for f in named if f[0] not in int8._TILES} - {"64_split"}
    assert few == {f"few{r}_c{c}" for r, c in ((16, 16), (16, 24), (16, 32), (16, 64), (32, 16), (32, 24), (32, 32), (64, 16),
                                               (64, 32))}
    for m, n, k in ((100, 1024, 4096), (150, 300, 16384), (64, 64, 16384), (70, 16, 131056)):
        steps, (splits, each) = -(-k // 128), int8._gemm_splits(m, n, k)
        assert int8._gemm_form(m, n, k)[0] == "64_split" and splits > 1 and (splits - 1) * each < steps <= splits * each
    for m in range(1, 65):
        kernel, rows, columns, threads = int8._gemm_form(m, 4096, 4096)
        assert rows >= m and columns % 8 == 0 and threads in (256, 512)


@pytest.mark.parametrize("d", [64, 128])
def test_attention_forms(d):
    forms = set()
    for heads, shared in ((1, 1), (8, 8), (8, 2), (32, 8), (30, 10)):
        for tokens in SIZES:
            for batch in (0, 1, 2, 8, 64, 1000):
                kind, rows, waves, two = form = packed._forward_form(heads, shared, tokens, batch, d)
                forms.add(form)
                assert not two or heads // shared % 2 == 0
                assert (kind == "_w8") == (waves == 8) and (kind == "_split") == (rows == 32)
    assert forms == {("_split", 32, 4, False), ("", 128, 4, False)} | (
        {("_w8", 128, 8, True), ("_w8", 256, 8, False)} if d == 128 else set())


@pytest.mark.parametrize("part", ["forward", "dq", "dkdv"])
def test_small_launches_divide(part):
    """One long sequence of few heads divides; many heads, and many short sequences, do not."""
    for d in (64, 128):
        assert packed._splits(part, 4, 1, 2048, 1, d)
        assert not packed._splits(part, 64, 1, 8192, 1, d)
        assert not packed._splits(part, 32, 1, 64 * 64, 64, d)


def test_threads_stay_below_the_launch_limit():
    """The largest call that passes the check, in the form with the most threads a token."""
    for tokens, batch, heads in (((1 << 23) // 8 * 128 - 128 * 300, 0, 8), (1 << 20, 0, 1000), (0, (1 << 23) // 8 - 2, 8)):
        assert (tokens // packed.ROWS + batch + 1) * heads < 1 << 23
        for part in ("forward", "dq", "dkdv"):
            for d in (64, 128):
                rows = 32 if packed._splits(part, heads, 1, tokens, batch, d) else 128
                assert (tokens // rows + batch + 1) * heads * 512 < 1 << 32
