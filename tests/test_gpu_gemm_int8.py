"""8-bit integer rows and their product.  Codes and scales follow from the
definition exactly.  A sum of products is exact, so an output's error is its
conversion and two products in fp32 (3 * 2^-24 of itself) and one rounding to
bf16 (2^-8): the same four roundings by torch give the same bits."""
import math

import pytest
import torch

from oracle.packed_ref import gemm_int8_ref, quantize_ref
from oracle.torch_ref import seeded_normal
from tests.conftest import announce
from warpir_amd import api, int8

pytestmark = pytest.mark.gpu


def _same_quantities(x, codes, scale):
    want, want_scale = quantize_ref(x.cpu())
    assert torch.equal(codes.cpu(), want)
    assert torch.equal(scale.cpu().nan_to_num(-1.0), want_scale.nan_to_num(-1.0))


@pytest.mark.parametrize("rows,width", [(1, 16), (5, 48), (3, 1024), (9, 1040), (2, 4096), (3, 4112), (2, 8192), (1, 8208),
                                        (2, 16384), (1, 16400), (1, 40000)])
def test_quantize(gpu, rows, width):
    announce(f"quantize {rows} x {width}")
    x = seeded_normal((rows, width + 24), 0, 3.0).cuda()[:, 8:width + 8]
    for _ in range(3):   # the call and its plan
        codes, scale = api.quantize_int8(x)
        _same_quantities(x, codes, scale)
    given = torch.full((rows, width + 32), 9, dtype=torch.int8, device="cuda")
    scale = torch.empty(rows, device="cuda")
    got = api.quantize_int8(x, codes=given[:, 16:width + 16], scale=scale)
    assert got[1] is scale and torch.equal(got[0], codes)
    assert bool((given[:, :16] == 9).all()) and bool((given[:, width + 16:] == 9).all())


def test_quantize_as_torch_divides(gpu):
    """Scales, and so codes, of a program that had them from torch on the GPU: bit for bit."""
    x = seeded_normal((4096, 256), 3).cuda()
    x[:, 0] = torch.arange(0x3f80, 0x3f80 + 4096, dtype=torch.int16, device="cuda").view(torch.bfloat16)   # every mantissa
    x[:, 1:] = x[:, 1:].clamp(-1, 1)
    codes, scale = api.quantize_int8(x)
    want = x.float().abs().amax(1) / 127
    assert torch.equal(scale, want)
    assert torch.equal(codes, (x.double() / want.double()[:, None]).round().to(torch.int8))


def test_quantize_borders(gpu):
    """Quotients on and next to the borders between codes, magnitudes from the smallest to the largest, what is no number."""
    tie = torch.arange(-127, 128).float()
    rows = [torch.cat((tie, tie[tie.abs() < 127] + 0.5, torch.zeros(4)))[:512 - 4] * 2.0 ** e for e in (-100, -3, 0, 90)]
    rows += [seeded_normal((508,), i).float() * 2.0 ** e for i, e in enumerate((-133, -130, -126, -119, -118, 0, 100, 125))]
    x = torch.zeros(len(rows) + 5, 512, dtype=torch.bfloat16)
    for i, row in enumerate(rows):
        x[i, :508] = row[:508].bfloat16() if row.numel() >= 508 else torch.nn.functional.pad(row, (0, 508 - row.numel())).bfloat16()
    x[len(rows)] = 0.0
    x[len(rows) + 1, 17] = 2.0 ** -133                 # the smallest bf16
    x[len(rows) + 2, 500] = torch.finfo(torch.bfloat16).max
    x[len(rows) + 3, 40], x[len(rows) + 3, 3] = math.inf, 2.0
    x[len(rows) + 4, 511] = math.nan
    codes, scale = api.quantize_int8(x.cuda())
    _same_quantities(x, codes, scale)


def _operands(m, n, k, seed=0):
    gen = torch.Generator().manual_seed(seed)
    a, b = (torch.randint(-128, 128, (r, k), generator=gen, dtype=torch.int8).cuda() for r in (m, n))
    return a, b, *((torch.rand(r, generator=gen) * 0.01 + 1e-4).cuda() for r in (m, n))


def _check(out, a, b, sa, sb):
    ref = gemm_int8_ref(*(t.cpu() for t in (a, b, sa, sb)))
    off = (out.cpu().double() - ref).abs()
    assert bool((off <= (2 ** -8 + 2 ** -21) * ref.abs()).all()), off.max()
    total = (a.cpu().double() @ b.cpu().double().T).float()   # rounded once, as the conversion of an integer is
    assert torch.equal(out.cpu(), (total * sa.cpu()[:, None] * sb.cpu()).bfloat16())


@pytest.mark.parametrize("m,n,k", [
    (1, 1, 16), (1, 16, 16), (1, 4096, 512), (3, 17, 144), (16, 300, 4096), (17, 64, 128), (32, 1000, 1040), (33, 31, 2064),
    (64, 512, 96), (65, 513, 272), (100, 4100, 528), (128, 128, 128), (300, 200, 1000 // 16 * 16), (777, 1030, 64),
    (1, 20, 131056), (200, 3000, 112)])
def test_gemm(gpu, m, n, k):
    announce(f"gemm int8 {m} x {n} x {k}")
    a, b, sa, sb = _operands(m, n, k)
    for _ in range(3):   # the call and its plan
        _check(api.gemm_int8(a, b, sa, sb), a, b, sa, sb)


@pytest.mark.parametrize("m,n,k", [(2048, 2048, 256), (2100, 1990, 400), (4096, 4352, 144), (4100, 4100, 512)])
def test_gemm_large_tiles(gpu, m, n, k):
    announce(f"gemm int8 {m} x {n} x {k}")
    a, b, sa, sb = _operands(m, n, k)
    _check(api.gemm_int8(a, b, sa, sb), a, b, sa, sb)


def test_gemm_extremes(gpu):
    """The largest sums of either sign, scales that give infinities, NaN and zeros, and the longest rows."""
    k = 131056
    a = torch.full((2, k), -128, dtype=torch.int8, device="cuda")
    b = torch.stack((torch.full((k,), -128, dtype=torch.int8), torch.full((k,), 127, dtype=torch.int8))).cuda()
    sa, sb = torch.tensor([1.0, 2.0 ** 90], device="cuda"), torch.tensor([1.0, 0.5], device="cuda")
    _check(api.gemm_int8(a, b, sa, sb), a, b, sa, sb)
    sa = torch.tensor([math.nan, 3e38], device="cuda")
    out = api.gemm_int8(a, b, sa, sb)
    assert bool(out[0].isnan().all()) and out[1].tolist() == [math.inf, -math.inf]


def test_gemm_views_and_results(gpu):
    m, n, k = 70, 90, 160
    wide = torch.randint(-128, 128, (m + n, k + 48), dtype=torch.int8, device="cuda")
    a, b = wide[:m, 16:k + 16], wide[m:, 32:k + 32]
    _, _, sa, sb = _operands(m, n, 16)
    want = api.gemm_int8(a.contiguous(), b.contiguous(), sa, sb)
    for _ in range(3):
        assert torch.equal(api.gemm_int8(a, b, sa, sb), want)
        for pad, at in ((6, 0), (11, 3), (38, 8)):     # rows that 16-byte stores fit, and that they do not
            big = torch.full((m, n + pad), 5.0, dtype=torch.bfloat16, device="cuda")
            out = big[:, at:at + n]
            assert api.gemm_int8(a, b, sa, sb, out=out) is out and torch.equal(out, want)
            assert bool((big[:, :at] == 5.0).all()) and bool((big[:, at + n:] == 5.0).all())
    assert api.gemm_int8(a[:0], b, sa[:0], sb).shape == (0, n) and api.gemm_int8(a, b[:0], sa, sb[:0]).shape == (m, 0)
    assert bool((api.gemm_int8(a[:, :0], b[:, :0], sa, sb) == 0).all())
    codes, scale = api.quantize_int8(torch.empty(0, 32, dtype=torch.bfloat16, device="cuda"))
    assert codes.shape == (0, 32) and scale.shape == (0,)
    assert torch.equal(api.gemm_int8(a, a, sa, sa), api.gemm_int8(a, a.clone(), sa, sa.clone()))


def test_streams_and_graphs(gpu):
    x = seeded_normal((40, 1024), 0).cuda()
    w, ws = api.quantize_int8(seeded_normal((520, 1024), 1).cuda())

    def step(x):
        return api.gemm_int8(*_order(api.quantize_int8(x), w, ws))

    want = step(x)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = step(x)
    side.synchronize()
    assert torch.equal(got, want)
    held = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(held)
    for n in range(4):
        held.copy_(x * (n + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, step(held))


def _order(rows, w, ws):
    return rows[0], w, rows[1], ws
