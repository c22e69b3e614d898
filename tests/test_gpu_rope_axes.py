"""The rotation by several axes against the 64-bit oracle.

Tolerance, derived: an output is rounded once to bf16, at most 2^-8 of itself;
before that the table's values (rounded once, 2^-24 of themselves, at most 1),
two products and a sum of at most |a| + |b|: 4 * 2^-24 (|a| + |b|)."""
import pytest
import torch

from oracle.packed_ref import axes_angles_ref, rope_axes_ref
from oracle.torch_ref import seeded_normal
from tests.conftest import announce
from warpir_amd import api

pytestmark = pytest.mark.gpu


def _check(got, x, angle, inter, back):
    ref, bound = rope_axes_ref(x.cpu(), angle, inter, back)
    off = (got.cpu().double() - ref).abs()
    assert bool((off <= 2 ** -8 * ref.abs() + 2 ** -22 * bound).all()), off.max()
    r = 2 * angle.shape[-1]
    assert torch.equal(got[..., r:], x[..., r:])


def _heads(b, h, hk, s, d, packed, seed):
    if packed:
        x = seeded_normal((b, s, h + 2 * hk, d), seed).cuda().permute(0, 2, 1, 3)
        return x[:, :h], x[:, h:h + hk]
    return seeded_normal((b, h, s, d), seed).cuda(), seeded_normal((b, hk, s, d), seed + 1).cuda()


CASES = [   # b, h, hk, s, d, sections, interleaved, packed, positions
    (1, 1, 1, 1, 64, (8,), False, False, "shared"),
    (1, 3, 1, 9, 64, (32,), True, True, "shared"),
    (2, 4, 2, 33, 128, (16, 24, 24), False, True, "each"),
    (1, 16, 4, 257, 128, (16, 24, 24), True, True, "wide"),
    (3, 2, 2, 17, 64, (4, 12), False, False, "each"),
    (1, 5, 1, 40, 128, (1, 2, 5, 0), True, True, "wide"),
    (1, 5, 1, 40, 128, (3, 30, 7, 16), False, True, "shared"),
    (2, 0, 3, 11, 64, (0, 8, 8), False, False, "wide"),
    (2, 3, 0, 11, 128, (5, 19), True, False, "each"),
    (1, 2, 1, 900, 64, (8, 8, 8), False, True, "strided"),
]


@pytest.mark.parametrize("b,h,hk,s,d,sections,inter,packed,where", CASES)
def test_forward_and_backward(gpu, b, h, hk, s, d, sections, inter, packed, where):
    announce(f"rope axes B{b} H{h}/{hk} S{s} D{d} {sections} inter={inter} packed={packed} {where}")
    rows, axes, pairs = 120, len(sections), sum(sections)
    gen = torch.Generator().manual_seed(3)
    pos = torch.randint(0, rows, (axes, 1 if where in ("shared", "strided") else b, s), generator=gen)
    freq = 100.0 ** (-torch.arange(pairs, dtype=torch.float64) / pairs)
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * freq
    wide = torch.zeros(2, rows, pairs + 4)
    wide[0, :, :pairs], wide[1, :, :pairs] = angle.cos().float(), angle.sin().float()
    cos, sin = (x[:, :pairs] for x in wide.cuda())
    given = (pos[:, 0] if where in ("shared", "strided") else pos).cuda()
    given = given.int() if where != "wide" else given
    if where == "strided":
        given = torch.stack((given, given + 1), -1)[..., 0]
    turned = axes_angles_ref(pos, freq, sections).expand(b, s, pairs)
    q, k = _heads(b, h, hk, s, d, packed, 0)
    gq, gk = _heads(b, h, hk, s, d, not packed, 5)
    for _ in range(3):   # the call and its plan
        got = api.rope_axes(q, k, cos, sin, given, sections, interleaved=inter)
        back = api.rope_axes_backward(gq, gk, cos, sin, given, list(sections), interleaved=inter)
        for x, y, way in ((got[0], q, False), (got[1], k, False), (back[0], gq, True), (back[1], gk, True)):
            assert x.is_contiguous()
            _check(x, y, turned, inter, way)


def test_frequencies_that_go_on(gpu):
    """With one position for every axis this is the rotation by one axis, whatever the sections."""
    q, k = _heads(1, 4, 2, 50, 128, True, 0)
    cos, sin = api.rope_table(64, 128)
    pos = (torch.arange(50, device="cuda") + 7).int()
    one = api.rope_axes(q, k, cos, sin, pos[None], (64,))
    many = api.rope_axes(q, k, cos, sin, pos.expand(3, 50), (10, 30, 24))
    assert all(torch.equal(a, b) for a, b in zip(one, many))
    _check(one[0], q, (pos.cpu().double()[:, None] * 10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64))[None], False, False)


@pytest.mark.parametrize("sections", [(8, 16), (6, 18)])
def test_positions_outside_the_table(gpu, sections):
    q, k = _heads(1, 2, 1, 6, 64, True, 0)
    cos, sin = api.rope_table(10, 48)
    pos = torch.tensor([[0, 9, 3, 4, 5, 6], [2, 3, 10, -1, 2 ** 31 - 1, -2 ** 31]], dtype=torch.int32, device="cuda")
    out, _ = api.rope_axes(q, k, cos, sin, pos, sections)
    n = sections[0]
    assert not bool(out[:, :, :2].isnan().any()) and not bool(out[..., 48:].isnan().any())
    assert bool(out[:, :, 2:, n:24].isnan().all()) and bool(out[:, :, 2:, 24 + n:48].isnan().all())
    assert not bool(out[..., :n].isnan().any()) and not bool(out[..., 24:24 + n].isnan().any())


def test_results_given(gpu):
    q, k = _heads(2, 4, 2, 19, 128, True, 0)
    cos, sin = api.rope_table(30, 96)
    pos = torch.randint(0, 30, (2, 2, 19), device="cuda")
    how = (cos, sin, pos, (20, 28))
    want = api.rope_axes(q, k, *how)
    for _ in range(3):
        x = torch.full((2, 19, 8, 128), 5.0, dtype=torch.bfloat16, device="cuda").permute(0, 2, 1, 3)
        got = api.rope_axes(q, k, *how, q_out=x[:, 1:5], k_out=x[:, 6:])
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and bool((x[:, [0, 5]] == 5.0).all())
        y = torch.cat((q, k), 1).permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
        got = api.rope_axes(y[:, :4], y[:, 4:], *how, q_out=y[:, :4], k_out=y[:, 4:])
        assert got[0].data_ptr() == y.data_ptr() and all(torch.equal(a, b) for a, b in zip(got, want))
        z = [t.clone() for t in want]
        assert api.rope_axes_backward(*z, *how, dq=z[0], dk=z[1])[0] is z[0]
        back = api.rope_axes_backward(*want, *how)
        assert all(torch.equal(a, b) for a, b in zip(z, back))
    with pytest.raises(ValueError, match="q_out and k have memory in common"):
        api.rope_axes(y[:, :2], y[:, 2:4], *how, q_out=y[:, 2:4])


def test_streams_and_graphs(gpu):
    q, k = _heads(1, 4, 2, 70, 64, True, 0)
    cos, sin = api.rope_table(100, 32)
    pos = torch.randint(0, 100, (2, 70), device="cuda", dtype=torch.int32)
    held = pos.clone()
    side = torch.cuda.Stream()
    want = api.rope_axes(q, k, cos, sin, pos, (8, 8))
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = api.rope_axes(q, k, cos, sin, pos, (8, 8))
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = api.rope_axes_backward(*api.rope_axes(q, k, cos, sin, held, (8, 8)), cos, sin, held, (8, 8))
    for n in range(4):
        held.copy_((pos + n) % 100)
        graph.replay()
        torch.cuda.synchronize()
        again = api.rope_axes_backward(*api.rope_axes(q, k, cos, sin, held, (8, 8)), cos, sin, held, (8, 8))
        assert all(torch.equal(a, b) for a, b in zip(got, again))
