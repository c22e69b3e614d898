"""Every form that a call of the packed operators or of the int8 product may take, at
the sizes where each can go wrong: what the rules choose at the sizes of the other
tests is only some of them.  The checks and their tolerances are those tests'."""
import math

import pytest
import torch

from tests import test_gpu_attention_packed as attention
from tests import test_gpu_gemm_int8 as product
from tests.conftest import announce
from warpir_amd import api, int8, packed
from warpir_amd.handwritten import DevicePlans

pytestmark = pytest.mark.gpu

FORMS = ["split", "four waves", "eight waves"]


@pytest.fixture
def take(monkeypatch):
    """Makes the calls take a form, in plans of their own."""
    def force(form):
        def forward(heads, shared, tokens, batch, d):
            if form == "split":
                return "_split", 32, 4, False
            if form == "eight waves" and d == 128:
                two = heads // shared % 2 == 0
                return "_w8", 128 if two else 256, 8, two
            return "", 128, 4, False

        monkeypatch.setattr(packed, "_forward_form", forward)
        monkeypatch.setattr(packed, "_splits", lambda *_: form == "split")
        monkeypatch.setattr(packed, "_forward_plans", DevicePlans("attention_packed"))
        monkeypatch.setattr(packed, "_backward_plans", DevicePlans("attention_packed_backward"))
    return force


MORE = [   # past the tests' own: two blocks of 256 rows and more, tiles that end inside every wave's rows
    (4, 2, 128, [1024, 257], 0, True),
    (3, 3, 128, [513, 255, 256], 300, True),
    (2, 2, 64, [1025], 3, False),
    (4, 1, 64, [260, 1000], 0, True),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("h,hk,d,lengths,rest,fused,form", [
    (*case, form) for case in attention.CASES + MORE for form in FORMS[:3 if case[2] == 128 else 2]])   # (D = 64: four waves only)
def test_forward_and_backward(gpu, take, form, h, hk, d, lengths, rest, fused, causal):
    announce(form)
    take(form)
    attention.test_forward_and_backward(gpu, h, hk, d, lengths, rest, fused, causal)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("d", [64, 128])
def test_scores(gpu, take, form, d):
    announce(form)
    take(form)
    attention.test_large_and_small_scores(gpu, d)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_what_a_row_does_not_see(gpu, take, form, value, d):
    announce(form)
    take(form)
    attention.test_what_a_row_does_not_see(gpu, value, d)
    attention.test_gradients_of_what_is_not_seen(gpu, value, d)


@pytest.mark.parametrize("form", FORMS)
def test_given_results_and_graphs(gpu, take, form):
    announce(form)
    take(form)
    attention.test_results_given(gpu)
    attention.test_offsets_that_are_none(gpu)
    attention.test_streams_and_graphs(gpu)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("batch", [62, 63, 64, 65, 510, 511, 512, 4200])
def test_many_sequences(gpu, take, form, batch):
    announce(form)
    take(form)
    attention.test_many_sequences(gpu, batch)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("batch", [3, 70, 600])
def test_offsets_that_do_not_ascend(gpu, take, form, batch):
    """They give wrong rows and no more: what lies beside the results stays."""
    announce(f"{form}, {batch} wild offsets")
    take(form)
    gen = torch.Generator().manual_seed(batch)
    t = 900
    offsets = torch.randint(-100, t + 100, (batch + 1,), generator=gen, dtype=torch.int32).cuda()
    q, k, v = attention._inputs(2, 1, 128, t, True)
    big = torch.full((t, 4, 128), 5.0, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    lse = torch.full((4, t), 7.0, device="cuda")
    o, l = api.attention_packed(q, k, v, offsets, out=big[1:3], lse=lse[1:3])
    do = attention.seeded_normal((2, t, 128), 3).cuda()
    grads = torch.full((t, 6, 128), 5.0, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    api.attention_packed_backward(q, k, v, o.nan_to_num(0.0), l.clamp(-50, 50), do, offsets, dq=grads[1:3], dk=grads[3:4], dv=grads[4:5])
    assert bool((big[[0, 3]] == 5.0).all()) and bool((lse[[0, 3]] == 7.0).all()) and bool((grads[[0, 5]] == 5.0).all())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("name", ["k", "v"])
def test_in_place_where_a_value_is_odd(gpu, take, name, d):
    """A pass over values that a row sees and that are no numbers is made again: out in q's place, dk in k's and dv in
    v's are read again by then."""
    ends = [0, 90, 400]
    for form in FORMS:
        announce(f"{form} D{d} {name}")
        take(form)
        q, k, v = attention._inputs(4, 2, d, ends[-1], True)
        do = attention.seeded_normal((ends[-1], 4, d), 7).cuda().transpose(0, 1)
        x = dict(k=k.clone(), v=v.clone())
        x[name][:, 200, 5] = math.nan
        offsets = torch.tensor(ends, dtype=torch.int32, device="cuda")
        want = api.attention_packed(q, x["k"], x["v"], offsets)
        grads = api.attention_packed_backward(q, x["k"], x["v"], *want, do, offsets)
        here = q.clone()
        got = api.attention_packed(here, x["k"], x["v"], offsets, out=here)
        dk, dv = x["k"].clone(), x["v"].clone()
        back = api.attention_packed_backward(q, dk, dv, *want, do, offsets, dk=dk, dv=dv)
        for a, b in zip((*got, *back), (*want, *grads)):
            assert torch.equal(a.nan_to_num(77.0), b.nan_to_num(77.0))


GEMM = [(t, *int8._TILES[t][:3]) for t in int8._TILES] + [
    (f"few{r}_c{c}", r, c, 64 * (4 if r == 64 or (r, c) == (32, 32) else 8))
    for r, c in ((16, 16), (16, 24), (16, 32), (16, 64), (32, 16), (32, 24), (32, 32), (64, 16), (64, 32))]


@pytest.mark.parametrize("parts", [1, 2, 3, 7, 16])
def test_gemm_divided(gpu, monkeypatch, parts):
    """Sums over parts of K, of one step of 128 and more, the last part shorter."""
    monkeypatch.setattr(int8, "_gemm_form", lambda m, n, k: ("64_split", 64, 64, 256))
    monkeypatch.setattr(int8, "_gemm_plans", DevicePlans("gemm_int8"))
    for m, n, k in ((1, 1, 16), (65, 3, 2000), (64, 64, 128 * 16), (130, 197, 6160), (100, 520, 128 * 33 + 16)):
        steps = -(-k // 128)
        each = -(-steps // min(parts, steps))
        monkeypatch.setattr(int8, "_gemm_splits", lambda m, n, k: (-(-steps // each), each))
        announce(f"gemm int8 {m} x {n} x {k} in {-(-steps // each)} parts")
        operands = product._operands(m, n, k, m + n)
        for _ in range(3):   # the call and its plan
            product._check(api.gemm_int8(*operands), *operands)
        wide = torch.full((m, n + 6), 5.0, dtype=torch.bfloat16, device="cuda")
        assert torch.equal(api.gemm_int8(*operands, out=wide[:, 3:n + 3]), api.gemm_int8(*operands))
        assert bool((wide[:, :3] == 5.0).all()) and bool((wide[:, n + 3:] == 5.0).all())


def test_gemm_divided_extremes(gpu):
    """The largest sums over parts of K, as the rules choose them."""
    k = 131056
    assert int8._gemm_form(66, 2, k)[0] == "64_split"
    a = torch.full((66, k), -128, dtype=torch.int8, device="cuda")
    b = torch.stack((torch.full((k,), -128, dtype=torch.int8), torch.full((k,), 127, dtype=torch.int8))).cuda()
    sa, sb = torch.full((66,), 2.0, device="cuda"), torch.tensor([1.0, 0.5], device="cuda")
    product._check(api.gemm_int8(a, b, sa, sb), a, b, sa, sb)


def test_gemm_divided_graphs(gpu):
    """Two graphs with a workspace each, replayed in turn with eager calls between them."""
    m, n, k = 150, 300, 4096
    assert int8._gemm_form(m, n, k)[0] == "64_split"
    held = [product._operands(m, n, k, seed) for seed in (1, 2)]
    want = [api.gemm_int8(*x) for x in held]
    graphs = []
    for x in held:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = api.gemm_int8(*x)
        graphs.append((graph, out))
    for i in range(6):
        graph, out = graphs[i % 2]
        graph.replay()
        got = api.gemm_int8(*held[1 - i % 2])
        torch.cuda.synchronize()
        assert torch.equal(out, want[i % 2]) and torch.equal(got, want[1 - i % 2])


@pytest.mark.parametrize("form", GEMM, ids=lambda f: f[0])
def test_gemm(gpu, monkeypatch, form):
    rows = form[1]
    monkeypatch.setattr(int8, "_gemm_form", lambda m, n, k: form)
    monkeypatch.setattr(int8, "_gemm_plans", DevicePlans("gemm_int8"))
    ms = [1, rows - 1, rows] + ([rows + 1, 2 * rows + 37] if form[0] in int8._TILES else [])
    sizes = [(m, n, k) for i, m in enumerate(ms) for n, k in ((1, 16), (form[2] + 3, 144), (2 * form[2] + 8, 1040 + 128 * i), (517, 400))]
    for m, n, k in sizes + [(rows, 9, 4112), (rows, form[2], 2048), (rows, form[2], 6160)]:
        announce(f"gemm int8 {form[0]} {m} x {n} x {k}")
        operands = product._operands(m, n, k, m + n)
        product._check(api.gemm_int8(*operands), *operands)
