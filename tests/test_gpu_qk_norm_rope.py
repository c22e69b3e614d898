"""The head norms with rotation and their gradients against the 64-bit oracle.

Tolerances, derived: an output is rounded once to bf16, at most 2^-8 of
itself.  Before that, in fp32: the mean square adds D positive terms in a
chain of at most 16 and 3 lane steps (19 roundings), the square root, the
division and the two products add 4, so a normed value is off by less than
2^-19 of itself; the rotation adds three roundings and the table's one of
each pair value.  2^-18 (|a| + |b|) bounds all of it.  A gradient is the same
with one more mean (2^-17 of the sum of its terms' magnitudes); a weight's
gradient adds at most a few hundred terms in a chain (2^-15 of the sum of
the terms' magnitudes)."""
import pytest
import torch

from oracle.layer_ref import angles_ref, norm_rope_bwd_ref, norm_rope_ref
from oracle.torch_ref import seeded_normal
from tests.conftest import announce
from warpir_amd import api, plans, rotary

pytestmark = pytest.mark.gpu


def _inputs(b, h, hk, s, d, packed, wide, seed=0):
    if packed:
        qkv = seeded_normal((b, s, h + 2 * hk, d), seed).cuda().permute(0, 2, 1, 3)
        q, k = qkv[:, :h], qkv[:, h:h + hk]
    else:
        q, k = seeded_normal((b, h, s, d), seed).cuda(), seeded_normal((b, hk, s, d), seed + 1).cuda()
    weights = [(1 + 0.3 * seeded_normal((d,), seed + 2 + i).float()).to(torch.float32 if wide else torch.bfloat16).cuda()
               for i in range(2)]
    return q, k, *weights


def _check(got, x, w, angle, inter, eps=1e-6):
    ref, size = norm_rope_ref(x.cpu(), w.cpu(), angle, eps, inter)
    off = (got.cpu().double() - ref).abs()
    assert bool((off <= 2 ** -8 * ref.abs() + 2 ** -18 * size).all()), off.max()


def _check_bwd(got, gw, g, x, w, angle, inter, eps=1e-6):
    dx, dw, size, size_w = norm_rope_bwd_ref(g.cpu(), x.cpu(), w.cpu(), angle, eps, inter)
    off = (got.cpu().double() - dx).abs()
    assert bool((off <= 2 ** -8 * dx.abs() + 2 ** -17 * size).all()), off.max()
    assert bool(((gw.cpu().double() - dw).abs() <= 2 ** -15 * size_w).all())


CASES = [   # b, h, hk, s, d, packed, fp32 weights, interleaved, positions
    (1, 1, 1, 1, 64, False, False, False, None),
    (2, 3, 1, 1, 128, True, False, True, "far"),
    (1, 8, 2, 33, 64, True, True, False, "rows"),
    (3, 5, 5, 17, 128, False, False, False, None),
    (2, 4, 1, 129, 128, True, True, True, "one"),
    (1, 0, 3, 9, 64, False, False, False, "rows"),
    (7, 24, 8, 61, 64, True, False, True, "far"),
    (2, 16, 4, 700, 128, True, False, False, "rows"),
]


@pytest.mark.parametrize("b,h,hk,s,d,packed,wide,inter,where", CASES)
def test_forward_and_backward(gpu, b, h, hk, s, d, packed, wide, inter, where):
    announce(f"norm+rope B{b} H{h}/{hk} S{s} D{d} packed={packed} wide={wide} inter={inter} {where}")
    q, k, qw, kw = _inputs(b, h, hk, s, d, packed, wide)
    table = api.rope_table(1 << 17 if where == "far" else 2 * s + 40, d)
    pos = torch.arange(s).expand(b, s)
    given = None
    if where == "one":
        pos = (torch.arange(s) * 2 + 3).expand(b, s)
        given = pos[0].cuda()
    elif where:
        first = torch.tensor([(1 << 17) - s - 3 * i for i in range(b)] if where == "far" else list(range(b)))
        pos = first[:, None] + torch.arange(s)
        given = (pos.int() if where == "rows" else pos).cuda()
    angle = angles_ref(pos, d)
    for _ in range(2):   # the call and its plan
        qo, ko = api.qk_norm_rope(q, k, qw, kw, *table, positions=given, interleaved=inter)
        assert qo.shape == q.shape and ko.is_contiguous()
        _check(qo, q, qw, angle, inter)
        _check(ko, k, kw, angle, inter)
    gq, gk = seeded_normal(q.shape, 7).cuda(), seeded_normal((b, s, hk, d), 8).cuda().transpose(1, 2)
    first = None
    for _ in range(2):
        got = api.qk_norm_rope_backward(gq, gk, q, k, qw, kw, *table, positions=given, interleaved=inter)
        _check_bwd(got[0], got[2], gq, q, qw, angle, inter)
        _check_bwd(got[1], got[3], gk, k, kw, angle, inter)
        assert first is None or all(torch.equal(x, y) for x, y in zip(got, first))
        first = got


def test_many_rows_take_turns(gpu):
    """More rows than workgroups hold at once; a weight's gradient is a long sum."""
    q, k, qw, kw = _inputs(2, 12, 4, 5000, 64, True, True)
    gq, gk = (seeded_normal(x.shape, 9).cuda() for x in (q, k))
    table = api.rope_table(5000, 64)
    angle = angles_ref(torch.arange(5000)[None], 64)
    got = api.qk_norm_rope_backward(gq, gk, q, k, qw, kw, *table)
    _check_bwd(got[0], got[2], gq, q, qw, angle, False)
    _check_bwd(got[1], got[3], gk, k, kw, angle, False)


def test_outputs_given_in_place_and_strided(gpu):
    q, k, qw, kw = _inputs(2, 4, 2, 19, 128, True, False)
    table = api.rope_table(32, 128)
    want = api.qk_norm_rope(q, k, qw, kw, *table)
    big = torch.full((2, 19, 8, 128), 5.0, dtype=torch.bfloat16, device="cuda").permute(0, 2, 1, 3)
    got = api.qk_norm_rope(q, k, qw, kw, *table, q_out=big[:, 1:5], k_out=big[:, 6:])
    assert got[0].data_ptr() == big[:, 1:5].data_ptr() and all(torch.equal(x, y) for x, y in zip(got, want))
    assert bool((big[:, [0, 5]] == 5.0).all())
    gq, gk = torch.randn_like(want[0]), torch.randn_like(want[1])
    grads = api.qk_norm_rope_backward(gq, gk, q, k, qw, kw, *table)
    ws = torch.empty(1025 * 128, device="cuda")
    own = [torch.empty(128, device="cuda") for _ in range(2)]
    again = api.qk_norm_rope_backward(gq, gk, q, k, qw, kw, *table, dq=gq, dk=gk, dq_weight=own[0], dk_weight=own[1],
                                      workspace=ws)
    assert again[0] is gq and again[2] is own[0] and all(torch.equal(x, y) for x, y in zip(again, grads))
    got = api.qk_norm_rope(q, k, qw, kw, *table, q_out=q, k_out=k)
    assert got[0] is q and all(torch.equal(x, y) for x, y in zip(got, want))


def test_in_place_and_one_weight_by_their_plans(gpu):
    """The results of calls with tensors of their own, and the tensors that were given."""
    q, k, w, _ = _inputs(2, 4, 2, 19, 64, True, False)
    table = api.rope_table(32, 64)
    want = api.qk_norm_rope(q, k, w, w.clone(), *table)
    gq, gk = torch.randn_like(want[0]), torch.randn_like(want[1])
    grads = api.qk_norm_rope_backward(gq, gk, q, k, w, w.clone(), *table)
    held = [[plans.native().size(p._table) for p in (rotary._forward_plans, rotary._backward_plans)]]
    for _ in range(3):
        x, y = q.clone(), k.clone()
        got = api.qk_norm_rope(x, y, w, w, *table, q_out=x, k_out=y)
        assert got[0] is x and got[1] is y and all(torch.equal(a, b) for a, b in zip(got, want))
        for over in ((gq, gk), (q, k)):
            at = [t.clone() for t in (gq, gk, q, k)]
            dq, dk = at[:2] if over[0] is gq else at[2:]
            got = api.qk_norm_rope_backward(*at, w, w, *table, dq=dq, dk=dk)
            assert got[0] is dq and got[1] is dk and all(torch.equal(a, b) for a, b in zip(got, grads))
        held.append([plans.native().size(p._table) for p in (rotary._forward_plans, rotary._backward_plans)])
    assert all(a < b for a, b in zip(*held[:2])) and held[1] == held[2] == held[3]


def test_positions_outside_the_table_and_special_rows(gpu):
    q, k, qw, kw = _inputs(1, 2, 1, 6, 64, False, False)
    q[0, 0, 3], q[0, 1, 4, 5], k[0, 0, 2, 1] = 0, float("inf"), float("nan")
    pos = torch.tensor([0, -1, 7, 8, 3, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    out, outk = api.qk_norm_rope(q, k, qw, kw, *api.rope_table(8, 64), positions=pos)
    bad = torch.tensor([False, True, False, True, False, True])
    assert bool(out[0, 0, bad].isnan().all()) and bool(out[0, 0, ~bad].isfinite().all())
    assert bool(outk[0, 0, 2].isnan().all()) and bool(outk[0, 0, [0, 4]].isfinite().all())
    assert bool(out[0, 1, 4].isnan().any())          # inf * rsqrt(inf)
    zero, _ = api.qk_norm_rope(torch.zeros_like(q), k, qw, kw, *api.rope_table(8, 64))
    assert bool((zero == 0).all())


def test_empty_rows(gpu):
    q = torch.empty(2, 3, 0, 64, dtype=torch.bfloat16, device="cuda")
    k, w = q[:, :1], torch.ones(64, dtype=torch.bfloat16, device="cuda")
    table = api.rope_table(4, 64)
    out = api.qk_norm_rope(q, k, w, w, *table)
    assert out[0].shape == q.shape and out[1].shape == k.shape
    grads = api.qk_norm_rope_backward(q, k, q, k, w, w, *table)
    assert bool((grads[2] == 0).all()) and bool((grads[3] == 0).all())


def test_streams_and_graphs(gpu):
    q, k, qw, kw = _inputs(2, 8, 2, 40, 128, False, False)
    gq, gk = seeded_normal(q.shape, 3).cuda(), seeded_normal(k.shape, 4).cuda()
    table = api.rope_table(64, 128)

    def step():
        return (*api.qk_norm_rope(q, k, qw, kw, *table), *api.qk_norm_rope_backward(gq, gk, q, k, qw, kw, *table))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(other, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for n in range(4):
        for x in (q, k, gq, gk):
            x.copy_(seeded_normal(x.shape, 20 + n).cuda())
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(held, step()))
