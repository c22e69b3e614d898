"""Attention over packed sequences and its gradients against the 64-bit oracle.

Tolerances, derived.  u = 2^-24 is half a step of fp32 relative to the value.
A score adds D exact products (bf16 by bf16) in fp32 and is multiplied by a
rounded constant: off by at most (D + 4) u S with S = sum |q_d k_d| / sqrt(D) (each
addition rounds a partial sum of at most S), so is the row's maximum, which both
numerator and denominator share; the exponential's argument is rounded (u times
its size, at most 2 S log2(e), and that of the running maximum) and the hardware's
exp2 and log2 are good to 2^-21.  e = 2 (D + 8) u S + 2^-20 bounds a probability's
relative error before it is rounded.  Sums over n keys round once a key at most,
and again for each of n / 64 tiles' new maxima: 2 n u.

O: one rounding to bf16 of the result (2^-8 of itself) and of each probability in
the product, but not in the sum below it (2^-8 of sum P |v|), and e and 2 n u of both.
LSE: e, 2 n u and the rounding of a number of its size, 4 u |LSE|.
Gradients: P comes from the LSE as it was given, so e holds with the LSE's size
in S's place as well; it is rounded for dV, dS for dQ and dK; the products of dO
with v and with O have errors of (D + 4) u of their magnitudes.  A probability (or
dS) below the smallest normal number, 2^-126 in bf16 as in fp32, may become 0:
each of n terms may lose 2^-126 times its other factors, which with these inputs
(values up to 6 * 6, D = 128 of them in a product) are less than 2^24."""
import math

import pytest
import torch

from oracle.packed_ref import packed_attention_bwd_ref, packed_attention_ref
from oracle.torch_ref import seeded_normal
from tests.conftest import announce
from warpir_amd import api

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _ends(lengths):
    ends = [0]
    for n in lengths:
        ends.append(ends[-1] + n)
    return ends


def _inputs(h, hk, d, t, fused, seed=0, scale=1.0):
    if fused:
        x = seeded_normal((t, h + 2 * hk, d), seed, scale).cuda().transpose(0, 1)
        return x[:h], x[h:h + hk], x[h + hk:]
    return [seeded_normal((n, t, d), seed + i, scale).cuda() for i, n in enumerate((h, hk, hk))]


def _longest(ends):
    return max([b - a for a, b in zip(ends, ends[1:])] + [0])


def _check_forward(o, lse, q, k, v, ends, causal):
    ref, ref_lse, weight, scores = packed_attention_ref(q.cpu(), k.cpu(), v.cpu(), ends, causal)
    n, d = _longest(ends), q.shape[-1]
    e = (2 * (d + 8) * U * scores + 2 ** -20)[..., None]
    off = (o.cpu().double() - ref).abs()
    assert bool((off <= 2 ** -8 * ref.abs() + (2 ** -8 + 2 * e + 4 * n * U) * weight).all()), off.max()
    lse = lse.cpu().double()
    assert torch.equal(lse.isinf(), ref_lse.isinf())
    fine = ~ref_lse.isinf()
    off = (lse - ref_lse)[fine].abs()
    assert bool((off <= (e[..., 0] + 2 * n * U)[fine] + 4 * U * ref_lse[fine].abs()).all()), off.max()


def _check_backward(grads, q, k, v, o, lse, do, ends, causal):
    refs, bounds, noise = packed_attention_bwd_ref(*(x.cpu() for x in (q, k, v, o, lse, do)), ends, causal)
    _, ref_lse, _, scores = packed_attention_ref(q.cpu(), k.cpu(), v.cpu(), ends, causal)
    n, d = _longest(ends), q.shape[-1]
    size = float((scores + torch.where(ref_lse.isinf(), 0.0, ref_lse.abs())).max()) if scores.numel() else 0.0
    e = 2 * (d + 8) * U * size + 2 ** -20
    n *= q.shape[0] // k.shape[0]
    for name, got, ref, bound, noisy in zip(("dq", "dk", "dv"), grads, refs, bounds, noise):
        off = (got.cpu().double() - ref).abs()
        tol = 2 ** -8 * ref.abs() + (2 ** -8 + 2 * e + 4 * n * U) * bound + n * 2 ** -102
        if name != "dv":
            tol += (d + 8) * U * noisy
        assert bool((off <= tol).all()), (name, (off - tol).max())


CASES = [   # h, hk, d, lengths, rest, fused projection
    (1, 1, 64, [1], 0, False),
    (2, 1, 128, [0, 1, 0, 2, 0], 0, True),
    (3, 3, 64, [63, 64, 65, 1, 128], 5, True),
    (4, 2, 128, [127, 128, 129, 31], 200, True),
    (8, 1, 64, [333, 40], 0, False),
    (4, 4, 128, [32, 33, 300, 0, 95, 97], 1, True),
    (6, 2, 64, [700], 0, True),
    (2, 2, 128, [577, 190], 130, False),
    (2, 1, 64, [5] * 70, 3, True),
    (1, 1, 128, [], 7, False),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("h,hk,d,lengths,rest,fused", CASES)
def test_forward_and_backward(gpu, h, hk, d, lengths, rest, fused, causal):
    announce(f"packed attention H{h}/{hk} D{d} {lengths[:6]} rest {rest} fused={fused} causal={causal}")
    ends = _ends(lengths)
    t = ends[-1] + rest
    q, k, v = _inputs(h, hk, d, t, fused)
    do = seeded_normal((t, h, d), 9).cuda().transpose(0, 1) if fused else seeded_normal((h, t, d), 9).cuda()
    offsets = torch.tensor(ends, dtype=torch.int32, device="cuda")
    first = None
    for _ in range(3):   # the call and its plan
        o, lse = api.attention_packed(q, k, v, offsets, causal=causal)
        assert o.shape == q.shape and o.transpose(0, 1).is_contiguous()
        assert bool((o[:, ends[-1]:] == 0).all()) and bool((lse[:, ends[-1]:] == -math.inf).all())
        grads = api.attention_packed_backward(q, k, v, o, lse, do, offsets, causal=causal)
        assert all(bool((g[:, ends[-1]:] == 0).all()) for g in grads)
        assert first is None or all(torch.equal(x, y) for x, y in zip((o, lse, *grads), first))
        first = (o, lse, *grads)
    _check_forward(o, lse, q, k, v, ends, causal)
    _check_backward(grads, q, k, v, o, lse, do, ends, causal)


@pytest.mark.parametrize("d", [64, 128])
def test_large_and_small_scores(gpu, d):
    """Rows ruled by one key, and rows of equal keys."""
    for scale in (6.0, 0.0):
        announce(f"packed attention D{d} values times {scale}")
        ends = _ends([150, 64, 77])
        q, k, v = _inputs(2, 1, d, ends[-1], True, scale=scale)
        v = seeded_normal(v.shape, 5).cuda()
        offsets = torch.tensor(ends, dtype=torch.int32, device="cuda")
        for causal in (True, False):
            o, lse = api.attention_packed(q, k, v, offsets, causal=causal)
            _check_forward(o, lse, q, k, v, ends, causal)
            do = seeded_normal(q.shape, 6).cuda()
            grads = api.attention_packed_backward(q, k, v, o, lse, do, offsets, causal=causal)
            _check_backward(grads, q, k, v, o, lse, do, ends, causal)


@pytest.mark.parametrize("batch", [63, 64, 100, 4095, 4096, 4200])
def test_many_sequences(gpu, batch):
    """More sequences than the lanes of a wave look at in one and in two rounds: every sequence as by itself."""
    announce(f"packed attention, {batch} sequences")
    gen = torch.Generator().manual_seed(batch)
    lengths = torch.randint(0, 6, (batch,), generator=gen).tolist()
    lengths[-1] = 3
    ends = _ends(lengths)
    q, k, v = _inputs(1, 1, 64, ends[-1] + 2, True)
    o, lse = api.attention_packed(q, k, v, torch.tensor(ends, dtype=torch.int32, device="cuda"))
    _check_forward(o, lse, q, k, v, ends, True)


def _poison(x, where, value):
    y = x.clone()
    y[:, where] = value
    return y


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_what_a_row_does_not_see(gpu, value, d):
    """An infinity or NaN in one token's k or v: rows before it, the other sequences and the rows
    behind them have their results bit for bit; rows that see it do not hide it."""
    ends, at = _ends([100, 200, 70]), 100 + 77
    q, k, v = _inputs(4, 2, d, ends[-1] + 10, True)
    offsets = torch.tensor(ends, dtype=torch.int32, device="cuda")
    tokens = torch.arange(ends[-1] + 10, device="cuda")
    for causal in (True, False):
        want = api.attention_packed(q, k, v, offsets, causal=causal)
        sees = (tokens >= (at if causal else 100)) & (tokens < 300)
        for name in ("k", "v"):
            announce(f"packed attention D{d} {name} of a token is {value}, causal={causal}")
            bad = _poison({"k": k, "v": v}[name], at, value)
            o, lse = api.attention_packed(q, bad if name == "k" else k, bad if name == "v" else v, offsets, causal=causal)
            assert torch.equal(o[:, ~sees], want[0][:, ~sees]) and torch.equal(lse[:, ~sees], want[1][:, ~sees])
            if name == "v" and not math.isnan(value):
                assert bool((o[:, sees] == value).all()) and torch.equal(lse, want[1])
            elif name == "v":
                assert bool(o[:, sees].isnan().all()) and torch.equal(lse, want[1])
            elif math.isnan(value):
                assert bool(o[:, sees].isnan().all()) and bool(lse[:, sees].isnan().all())
    # both infinities in a column: rows that see one of them, and both
    bad = _poison(_poison(v, at, math.inf), at + 9, -math.inf)
    o = api.attention_packed(q, k, bad, offsets)[0]
    assert bool((o[:, at:at + 9] == math.inf).all()) and bool(o[:, at + 9:300].isnan().all())
    # what lies behind the last sequence is no one's
    rest = [_poison(x, slice(ends[-1], None), value) for x in (q, k, v)]
    o, lse = api.attention_packed(*rest, offsets)
    want = api.attention_packed(q, k, v, offsets)
    assert torch.equal(o, want[0]) and torch.equal(lse, want[1])


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_gradients_of_what_is_not_seen(gpu, value, d):
    """One token's q, k, v or dO is infinite or NaN: the gradients that do not depend on it are as they were."""
    ends, at = _ends([100, 200, 70]), 100 + 77
    q, k, v = _inputs(4, 2, d, ends[-1], True)
    do = seeded_normal((ends[-1], 4, d), 7).cuda().transpose(0, 1)
    offsets = torch.tensor(ends, dtype=torch.int32, device="cuda")
    o, lse = api.attention_packed(q, k, v, offsets)
    want = api.attention_packed_backward(q, k, v, o, lse, do, offsets)
    tokens = torch.arange(ends[-1], device="cuda")
    later, earlier = (tokens >= at) & (tokens < 300), (tokens <= at) & (tokens >= 100)
    other = (tokens < 100) | (tokens >= 300)
    for name in ("q", "k", "v", "do"):
        announce(f"packed attention backward D{d}, {name} of a token is {value}")
        x = dict(q=q, k=k, v=v, do=do)
        x[name] = _poison(x[name], at, value)
        o, lse = api.attention_packed(x["q"], x["k"], x["v"], offsets)
        dq, dk, dv = api.attention_packed_backward(x["q"], x["k"], x["v"], o, lse, x["do"], offsets)
        for got, ref in zip((dq, dk, dv), want):
            assert torch.equal(got[:, other], ref[:, other])
        if name in ("k", "v"):     # rows before the token do not see it, and those from it on are not numbers
            assert torch.equal(dq[:, ~later], want[0][:, ~later])
            if name == "v" or math.isnan(value):
                assert bool(dq[:, later].isnan().all())
        else:                      # one row's: keys after it are not seen by it
            assert torch.equal(dq[:, tokens != at], want[0][:, tokens != at])
            for got, ref in ((dk, want[1]), (dv, want[2])):
                assert torch.equal(got[:, ~earlier], ref[:, ~earlier])
            if math.isnan(value):
                assert bool(dk[:, earlier].isnan().all()) and bool(dv[:, earlier].isnan().all())


def test_results_given(gpu):
    """Rows of no sequence stay, results with strides, results in place."""
    h, hk, d, ends = 4, 2, 128, _ends([40, 0, 133])
    t = ends[-1] + 30
    q, k, v = _inputs(h, hk, d, t, True)
    do = seeded_normal((t, h, d), 7).cuda().transpose(0, 1)
    offsets = torch.tensor(ends, dtype=torch.int32, device="cuda")
    want = api.attention_packed(q, k, v, offsets)
    grads = api.attention_packed_backward(q, k, v, *want, do, offsets)
    for _ in range(3):
        out = torch.full((t, h + 1, d), 5.0, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
        lse = torch.full((t, h + 2), 7.0, device="cuda").t()
        got = api.attention_packed(q, k, v, offsets, out=out[1:], lse=lse[1:-1])
        assert got[0].data_ptr() == out[1:].data_ptr() and bool((out[0] == 5.0).all())
        assert torch.equal(got[0][:, :ends[-1]], want[0][:, :ends[-1]]) and bool((out[:, ends[-1]:] == 5.0).all())
        assert torch.equal(got[1][:, :ends[-1]], want[1][:, :ends[-1]]) and bool((lse[:, ends[-1]:] == 7.0).all())
        assert bool((lse[[0, -1]] == 7.0).all())
        # the projection's gradient in its own layout
        fused = torch.full((t, h + 2 * hk, d), 3.0, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
        ws = torch.empty(2 * h * t, device="cuda")
        got = api.attention_packed_backward(q, k, v, *want, do, offsets, dq=fused[:h], dk=fused[h:h + hk], dv=fused[h + hk:],
                                            workspace=ws)
        assert all(torch.equal(x[:, :ends[-1]], y[:, :ends[-1]]) for x, y in zip(got, grads))
        assert bool((fused[:, ends[-1]:] == 3.0).all())
        # in place of what is read by the same workgroup only
        x = torch.cat((q, k, v)).transpose(0, 1).contiguous().transpose(0, 1)
        xq, xk, xv = x[:h], x[h:h + hk], x[h + hk:]
        got = api.attention_packed(xq, xk, xv, offsets, out=xq)
        assert got[0] is xq and torch.equal(xq[:, :ends[-1]], want[0][:, :ends[-1]])
        assert torch.equal(xq[:, ends[-1]:], q[:, ends[-1]:])
        got = api.attention_packed_backward(q, xk, xv, *want, do, offsets, dk=xk, dv=xv)
        assert got[1] is xk and all(torch.equal(a[:, :ends[-1]], b[:, :ends[-1]]) for a, b in zip(got, grads))
    for bad in (k, v[:, 3:33], q[1:]):
        big = torch.empty(0, device="cuda") if bad is None else bad
        with pytest.raises(ValueError, match="have memory in common|must have shape"):
            api.attention_packed(q, k, v, offsets, out=big)
    with pytest.raises(ValueError, match="dq and q have memory in common"):
        api.attention_packed_backward(q, k, v, *want, do, offsets, dq=q)


def test_one_tensor_for_keys_and_values(gpu):
    ends = _ends([50, 20])
    q, k, _ = _inputs(2, 2, 64, ends[-1], False)
    offsets = torch.tensor(ends, dtype=torch.int32, device="cuda")
    want = api.attention_packed(q, k, k.clone(), offsets)
    got = api.attention_packed(q, k, k, offsets)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_offsets_that_are_none(gpu):
    """Offsets past the tokens end there, a first offset leaves what is before it, and a batch without tokens has
    empty results."""
    q, k, v = _inputs(2, 1, 64, 300, True)
    o = torch.full((2, 300, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    api.attention_packed(q, k, v, torch.tensor([140, 250, 900], dtype=torch.int32, device="cuda"), out=o)
    want = api.attention_packed(q, k, v, torch.tensor([0, 140, 250, 300], dtype=torch.int32, device="cuda"))[0]
    assert bool((o[:, :140] == 5.0).all()) and torch.equal(o[:, 140:], want[:, 140:])
    empty = [x[:, :0] for x in (q, k, v)]
    zero = torch.zeros(3, dtype=torch.int32, device="cuda")
    o, lse = api.attention_packed(*empty, zero)
    assert o.shape == (2, 0, 64) and lse.shape == (2, 0)
    assert [x.shape[1] for x in api.attention_packed_backward(*empty, o, lse, o.clone(), zero)] == [0, 0, 0]


def test_streams_and_graphs(gpu):
    """Side streams, two graphs of one shape, and replays over offsets that change."""
    h, hk, d, t = 4, 2, 64, 600
    q, k, v = _inputs(h, hk, d, t, True)
    do = seeded_normal((t, h, d), 7).cuda().transpose(0, 1)
    batches = [torch.tensor(x, dtype=torch.int32, device="cuda")
               for x in ([0, 200, 420, 600], [0, 1, 2, 3], [0, 0, 600, 600], [0, 300, 400, 555])]
    offsets = batches[0].clone()

    def step(at):
        o, lse = api.attention_packed(q, k, v, at)
        return (o, lse, *api.attention_packed_backward(q, k, v, o, lse, do, at))

    want = [step(x) for x in batches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s, x in zip(streams, batches):
        with torch.cuda.stream(s):
            s.wait_stream(torch.cuda.default_stream())
            got = step(x)
        s.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[0 if x is batches[0] else 1]))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step(offsets)
        graphs.append((graph, held))
    for n, x in enumerate(batches * 2):
        offsets.copy_(x)
        graph, held = graphs[n % 2]
        graph.replay()
        torch.cuda.synchronize()
        eager = step(x)
        assert all(torch.equal(a, b) for a, b in zip(held, want[n % len(batches)])), n
        assert all(torch.equal(a, b) for a, b in zip(eager, want[n % len(batches)])), n
