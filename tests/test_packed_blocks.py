"""Which rows the workgroups over packed sequences take, restated from
csrc/wir_packed.h (packed_block, packed_program) with its integer arithmetic: every
row of every sequence once, in whatever order the programs come, and rows within the tokens
for any offsets at all."""
import random

import pytest


def _offset(offsets, i, batch, tokens):
    return tokens if i > batch else min(max(offsets[i], 0), tokens)


def packed_block(offsets, batch, tokens, x, rows):
    """(start, len, row0, rest) of block x; each offset is read within the offsets."""
    lo, n = 0, batch + 1
    while True:
        step = (n + 63) // 64
        last = 0
        for lane in range(64):
            i = lo + lane * step
            at = _offset(offsets, min(i, batch), batch, tokens)
            if lane * step < n and at // rows + i <= x:
                last = lane
        if step > 1:
            lo, n = lo + last * step, min(step, n - last * step)
            continue
        seq = lo + last
        start, end = (_offset(offsets, min(seq, batch) + j, batch, tokens) for j in (0, 1))
        return start, end - start, (x - start // rows - seq) * rows, seq == batch


def place(x, blocks, tokens, batch, rows):
    """Program x's block of a head."""
    one = rows * batch
    if 4 * tokens > 3 * one and 2 * tokens < 3 * one and (x | 63) < blocks:
        return x & ~63 | (x & 31) << 1 | x >> 5 & 1
    return x


@pytest.mark.parametrize("rows", [32, 128, 256])
def test_every_block_once(rows):
    """The order of the programs is a permutation, for every number of blocks up to some hundreds and larger odd ones."""
    moved = 0
    for batch in [*range(1, 200), 511, 512, 1000, 4097]:
        for tokens in (rows * batch, rows * batch * 3 // 4 + 1, rows * batch * 3 // 2 - 1, rows * batch // 2, 2 * rows * batch):
            blocks = tokens // rows + batch + 1
            order = [place(x, blocks, tokens, batch, rows) for x in range(blocks)]
            assert sorted(order) == list(range(blocks))
            moved += order != list(range(blocks))
    assert moved > 100


@pytest.mark.parametrize("rows", [32, 128, 256])
@pytest.mark.parametrize("batch", [0, 1, 2, 7, 62, 63, 64, 70, 130])
def test_every_row_once(batch, rows):
    rng = random.Random(batch * 1000 + rows)
    for longest in (1, rows // 2, rows, 2 * rows + 1, 5 * rows):
        ends = [0]
        for _ in range(batch):
            ends.append(ends[-1] + rng.choice((0, 1, longest, rng.randint(0, longest))))
        tokens = ends[-1] + rng.choice((0, 1, 300))
        blocks = tokens // rows + batch + 1
        seen = [0] * tokens
        for x in range(blocks):
            start, length, row0, rest = packed_block(ends, batch, tokens, place(x, blocks, tokens, batch, rows), rows)
            if not 0 <= row0 < length:
                continue
            assert not rest or start == ends[-1]
            for row in range(start + row0, start + min(row0 + rows, length)):
                seen[row] += 1
                assert rest == (row >= ends[-1])
        assert seen == [1] * tokens


@pytest.mark.parametrize("rows", [32, 128, 256])
@pytest.mark.parametrize("batch", [1, 3, 70, 600])
def test_wild_offsets_stay_inside(batch, rows):
    """Offsets that do not ascend, or lie outside the tokens: a block that works at all has a sequence inside them."""
    rng = random.Random(batch + rows)
    for tokens in (1, 33, 900, 5000):
        for wild in (100, 1 << 30):
            offsets = [rng.randint(-wild, tokens + wild - 1) if rng.random() < 0.7 else rng.randint(0, tokens) for _ in range(batch + 1)]
            blocks = tokens // rows + batch + 1
            for x in {*range(min(blocks, 40)), *(rng.randrange(blocks) for _ in range(40)), blocks - 1}:
                start, length, row0, rest = packed_block(offsets, batch, tokens, x, rows)
                if 0 <= row0 < length:
                    assert 0 <= start and start + length <= tokens and start + min(row0 + rows, length) <= tokens
                assert abs(row0) < 1 << 31
