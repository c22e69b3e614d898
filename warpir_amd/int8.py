"""Products in 8-bit integers: tokens' codes and scales, and the product of two
matrices of them (``csrc/gemm_int8.hip``)."""
from __future__ import annotations

import ctypes
import functools
from typing import Tuple

from warpir_amd.handwritten import DevicePlans, apart, check_tensor, check_written, launch, need

_quantize_plans = DevicePlans("quantize_int8")
_gemm_plans = DevicePlans("gemm_int8")

MAX_WIDTH = 131056   # 2^7 * 2^7 * 131056 < 2^31: a sum of that many products fits


class _QuantizeArgs(ctypes.Structure):
    _fields_ = [("x", ctypes.c_void_p), ("codes", ctypes.c_void_p), ("scale", ctypes.c_void_p),
                ("xs", ctypes.c_longlong), ("cs", ctypes.c_longlong), ("rows", ctypes.c_int), ("width", ctypes.c_int)]


class _Args(ctypes.Structure):
    _fields_ = [*((n, ctypes.c_void_p) for n in ("a", "b", "a_scale", "b_scale", "out", "partial")),
                *((n, ctypes.c_longlong) for n in ("as_", "bs", "os")), *((n, ctypes.c_int) for n in ("m", "n", "k", "splits", "each"))]


def _pitch(t) -> int:
    """Elements from a row to the next."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def quantize_int8(x, codes=None, scale=None) -> Tuple[object, object]:
    """The rows of ``x`` ``[M, K]`` (bf16, K a multiple of 16, 16-byte aligned rows) in
    8-bit integers: ``(codes, scale)``, int8 ``[M, K]`` and fp32 ``[M]``.  A row's scale is
    its largest magnitude times 1 / 127, each rounded to fp32 (as torch's ``amax(1) / 127``
    on a GPU; 2^-126 at least), its codes the integers nearest to ``x / scale``, ties to
    even: -127 to 127.  The scale of a row with an infinity or NaN is NaN, and its
    codes are 0.  Made for ``gemm_int8``: of tokens, and of a weight's channels where
    they are rows.  ``codes`` and ``scale`` share no memory with one another or with ``x``."""
    import torch

    fn, done = "quantize_int8", None
    if codes is not None or scale is not None:
        apart(fn, ("codes", "scale", "codes", "x", "scale", "x"), 3, codes, scale, codes, x, scale, x)
    done = _quantize_plans.run(0, x, codes, scale)
    if done is not None and done is not False:
        return done
    check_tensor(fn, "x", x, torch.bfloat16, (None, None), None)
    (rows, width), device = x.shape, x.device
    need(fn, width % 16 == 0 and 0 < width <= MAX_WIDTH, f"K must be a multiple of 16 up to {MAX_WIDTH}, got {width}")
    need(fn, rows < 1 << 24, "2^24 rows or more in one call")
    if codes is not None:
        check_tensor(fn, "codes", codes, torch.int8, (rows, width), device)
        check_written(fn, "codes", codes)
    if scale is not None:
        check_tensor(fn, "scale", scale, torch.float32, (rows,), device, rows=False)
        need(fn, rows <= 1 or scale.stride(0) == 1, "scale must be contiguous")
    rec = _quantize_plans.recording(done, x, codes, scale)
    if codes is None:
        codes = rec.alloc(torch.empty(rows, width, dtype=torch.int8, device=device))
    if scale is None:
        scale = rec.alloc(torch.empty(rows, dtype=torch.float32, device=device))
    if rows == 0:
        return codes, scale
    name, each = _quantize_form(width)
    launch(rec, device, "gemm_int8.hsaco", f"wir_quantize_int8_{name}", (-(-rows // each), 1, 1), (256, 1, 1),
           _QuantizeArgs(None, None, None, _pitch(x), _pitch(codes), rows, width), {"x": x, "codes": codes, "scale": scale})
    if rec:
        _quantize_plans.add(0, rec, codes, scale)
    return codes, scale


def _quantize_form(width: int) -> Tuple[str, int]:
    """(kernel, rows of a workgroup): a wave a row up to 1024 values, four past that, each lane with one, two or
    four times 16 values in registers."""
    if width <= 1024:
        return "w1", 4
    return "w4" if width <= 4096 else "w4_n2" if width <= 8192 else "w4_n4", 1


def gemm_int8(a, b, a_scale, b_scale, out=None):
    """``out[m, n] = sum_k a[m, k] b[n, k] * a_scale[m] * b_scale[n]`` (bf16 ``[M, N]``) of
    int8 ``a`` ``[M, K]`` (tokens, as ``quantize_int8`` gives them) and ``b`` ``[N, K]`` (a
    weight, channel by channel), scales fp32 ``[M]`` and ``[N]``.  K is a multiple of 16
    up to 131056, rows are 16-byte aligned; M and N are any.  The sum is exact in
    32-bit integers; it is converted, scaled and rounded to bf16 once each."""
    import torch

    fn, done = "gemm_int8", None
    if out is not None:
        apart(fn, ("out", "a", "out", "b", "out", "a_scale", "out", "b_scale"), 4, out, a, out, b, out, a_scale, out, b_scale)
    done = _gemm_plans.run(0, a, b, a_scale, b_scale, out)
    if done is not None and done is not False:
        return done
    check_tensor(fn, "a", a, torch.int8, (None, None), None)
    (m, k), device = a.shape, a.device
    check_tensor(fn, "b", b, torch.int8, (None, k), device)
    n = b.shape[0]
    need(fn, k % 16 == 0 and k <= MAX_WIDTH, f"K must be a multiple of 16 up to {MAX_WIDTH}, got {k}")
    for name, s, rows in (("a_scale", a_scale, m), ("b_scale", b_scale, n)):
        check_tensor(fn, name, s, torch.float32, (rows,), device, rows=False)
        need(fn, rows <= 1 or s.stride(0) == 1, f"{name} must be contiguous")
    for name, t in (("a", a), ("b", b)):
        need(fn, _pitch(t) < 1 << 23, f"{name}'s rows are 2^23 bytes or more apart")
    need(fn, max(m, n) < 1 << 30, "2^30 rows or more in one call")
    if out is not None:
        check_tensor(fn, "out", out, torch.bfloat16, (m, n), device, rows=False)
        need(fn, n <= 1 or m == 0 or out.stride(1) == 1, "out's last dimension must be contiguous")
        check_written(fn, "out", out)
    rec = _gemm_plans.recording(done, a, b, a_scale, b_scale, out)
    if out is None:
        out = rec.alloc(torch.empty(m, n, dtype=torch.bfloat16, device=device))
    if m == 0 or n == 0:
        return out
    if k == 0:   # (0 times a scale, which may be infinite or NaN)
        return out.copy_(a_scale[:, None] * 0.0 * b_scale)
    variant, bm, bn, threads = _gemm_form(m, n, k)
    tiles = -(-m // bm) * -(-n // bn)
    need(fn, tiles * threads < 1 << 32, "2^32 threads or more in one call")
    tensors = {"a": a, "b": b, "a_scale": a_scale, "b_scale": b_scale, "out": out}
    splits, each = _gemm_splits(m, n, k) if variant == "64_split" else (1, 0)
    args = _Args(*[None] * 6, _pitch(a), _pitch(b), _pitch(out), m, n, k, splits, each)
    if variant == "64_split":
        tensors["partial"] = rec.alloc(torch.empty(splits * tiles * bm * bn, dtype=torch.int32, device=device))
    launch(rec, device, "gemm_int8.hsaco", f"wir_gemm_int8_{variant}", (splits * tiles, 1, 1), (threads, 1, 1), args, tensors)
    if variant == "64_split":
        launch(rec, device, "gemm_int8.hsaco", "wir_gemm_int8_join", (tiles, 1, 1), (threads, 1, 1), args, tensors)
    if rec:
        _gemm_plans.add(0, rec, out)
    return out


# Tiles: rows and columns of a workgroup's output, its threads, how many workgroups a CU holds, and the time of a product
# in microseconds: fixed + per_m * M N / 1e6 + steps of 128 along K * step, where a launch of P programs on 256 CUs, R
# rounds of them and a rest r (of 1), has
#   step = light + busy * r                                  R = 0, or one whole round
#        = full * R, plus the same line from light to full for the rest.
# Least-squares fits (rms 4-8% in log time) to 33 products from 65 x 640 x 1680 to 8192 x 8192 x 8192; the tile with the
# smallest estimate was within 0.7% (geometric mean; 14% at worst) of the fastest.
_TILES = {
    "256": (256, 256, 512, 1, (7.14, 1.242, 0.302, 1.785, 0.339)),
    "256x128": (256, 128, 512, 1, (4.42, 0.833, 0.137, 1.092, 0.333)),
    "128_w4": (128, 128, 256, 2, (2.69, 0.816, 0.342, 1.234, 0.127)),
    "128": (128, 128, 512, 1, (4.35, 0.519, 0.0, 0.631, 0.620)),
    "128x64": (128, 64, 256, 2, (3.62, 0.447, 0.135, 0.717, 0.421)),
    "64": (64, 64, 256, 2, (3.52, 0.311, 0.094, 0.446, 0.920)),
}


def _estimate(tile: str, m: int, n: int, k: int, splits: int = 1) -> float:
    bm, bn, _, held, (fixed, light, busy, full, per_mn) = _TILES[tile]
    programs = -(-m // bm) * -(-n // bn) * splits
    rounds, rest = divmod(programs, 256 * held)
    rest /= 256 * held
    if rounds == 0 or (rounds == 1 and rest == 0):
        step = light + busy * (rounds + rest)
    else:
        step = full * rounds + (light + (full - light) * rest if rest else 0.0)
    us = fixed + -(--(-k // 128) // splits) * step
    return us + per_mn * 1e-6 * m * n if splits == 1 else us + 1.78 + 0.323 * splits + 0.00816 * programs


@functools.lru_cache(maxsize=1024)
def _gemm_splits(m: int, n: int, k: int) -> Tuple[int, int]:
    """(parts, steps of 128 of one) of a product whose K is divided: at most what a round of workgroups holds.

    us by parts: 150 x 300 x 16384 1 45.0, 2 26.6, 4 17.2, 8 13.8, 16 14.9; 100 x 1024 x 4096 14.1, 11.6, 10.3, 11.2,
    15.4; 512 x 512 x 8192 23.9, 17.2, 14.1, 17.1, 24.3; 512 x 512 x 2048 8.9, 9.7, 10.1, 14.6; 200 x 4096 x 4096 14.4, 17.1."""
    steps, tiles = -(-k // 128), -(-m // 64) * -(-n // 64)
    splits = min((s for s in (1, 2, 3, 4, 6, 8, 12, 16) if s <= steps and (s == 1 or s * tiles <= 512)),
                 key=lambda s: _estimate("64", m, n, k, s))
    each = -(-steps // splits)
    return -(-steps // each), each


@functools.lru_cache(maxsize=1024)
def _gemm_form(m: int, n: int, k: int) -> Tuple[str, int, int, int]:
    """(kernel, rows and columns of a workgroup's output, its threads).

    Up to 64 tokens the weight's bytes count, and the tokens' that every
    workgroup reads again: each takes 16 to 64 channels, so that as many as 256
    CUs have one, and its waves divide K.  us, 16 / 24 / 32 / 64 channels a
    workgroup, 16 tokens: N = 4096, K = 4096 6.2 / 6.6 / 6.7 / 8.8, 6144 x 4096 8.8 / 7.4 /
    7.8 / 9.3, 8192 x 8192 16.1 / 18.3 / 13.6 / 16.9, 32768 x 4096 36.8 / 35.0 / 33.3 / 29.5 (64 x 64
    tiles 14.8, 15.1, 27.2, 31.9); 64 tokens, 16 / 32 channels: 4096 x 4096 8.4 / 10.0, 8192 x 8192
    25.3 / 19.1 (tiles 15.4, 27.2).

    Few tiles of 64 x 64 with a long K are divided along it, and a second kernel
    joins the sums (`_gemm_splits`); with up to 4096 channels for 33 to 64 tokens too (us,
    undivided / divided: 64 x 1024, K = 4096 7.2 / 9.8, 8192 about 11.5 / 12, 16384 20.8 / 14.1)."""
    splits = _gemm_splits(m, n, k)[0]
    divided = _estimate("64", m, n, k, splits) if splits > 1 else float("inf")
    if 32 < m <= 64 and n <= 4096 and divided < 2.9 + 0.14 * -(-k // 128):
        return "64_split", 64, 64, 256
    if m <= 64:
        rows = 16 if m <= 16 else 32 if m <= 32 else 64
        columns = 16 if n <= 4096 else 24 if n <= 6144 and rows < 64 else 64 if n >= 16384 and rows == 16 else 32
        waves = 4 if rows == 64 or (rows, columns) == (32, 32) else 8
        return f"few{rows}_c{columns}", rows, columns, 64 * waves
    tile = min(_TILES, key=lambda t: _estimate(t, m, n, k))
    if divided < _estimate(tile, m, n, k):
        return "64_split", 64, 64, 256
    return (tile, *_TILES[tile][:3])


__all__ = ["quantize_int8", "gemm_int8"]
