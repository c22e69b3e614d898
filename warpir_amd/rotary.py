"""Head norms with position rotation: what lies between a fused projection
(``api.gemm``) and attention (``csrc/qk_norm_rope.hip``)."""
from __future__ import annotations

import ctypes
import functools
import struct
from typing import Optional, Tuple

from warpir_amd.handwritten import INT_MAX, DevicePlans, apart, check_tensor, check_written, launch, need, own

_forward_plans = DevicePlans("qk_norm_rope")
_backward_plans = DevicePlans("qk_norm_rope_backward")


class _Side(ctypes.Structure):
    _fields_ = [("x", ctypes.c_void_p), ("g", ctypes.c_void_p), ("out", ctypes.c_void_p), ("w", ctypes.c_void_p),
                *((n, ctypes.c_longlong) for n in ("xb", "xh", "xs", "gb", "gh", "gs", "ob", "oh", "os")),
                ("heads", ctypes.c_int), ("blocks", ctypes.c_int)]


class _Args(ctypes.Structure):
    _fields_ = [("q", _Side), ("k", _Side), ("cos", ctypes.c_void_p), ("sin", ctypes.c_void_p),
                ("pos", ctypes.c_void_p), ("partial", ctypes.c_void_p),
                *((n, ctypes.c_longlong) for n in ("pb", "ps", "cs", "ss")),
                ("batch", ctypes.c_int), ("seq", ctypes.c_int), ("table_rows", ctypes.c_int), ("flags", ctypes.c_int),
                ("eps", ctypes.c_float)]


class _GradArgs(ctypes.Structure):
    _fields_ = [("partial", ctypes.c_void_p), ("q", ctypes.c_void_p), ("k", ctypes.c_void_p),
                ("q_blocks", ctypes.c_int), ("k_blocks", ctypes.c_int), ("d", ctypes.c_int)]


def rope_table(positions: int, d: int, base: float = 10000.0, device="cuda"):
    """``(cos, sin)`` of ``pos * base ** (-2 i / d)`` for positions
    ``0 .. positions - 1`` and pairs ``i < d / 2``: fp32, rounded once from 64
    bits (an fp32 angle of a far position is off by 2^-24 of itself, 0.06
    radians at a million)."""
    import torch

    need("rope_table", positions > 0 and d > 0 and d % 2 == 0 and base > 0, "positions, an even d and a positive base")
    freq = base ** (-torch.arange(0, d, 2, dtype=torch.float64, device=device) / d)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


@functools.lru_cache(maxsize=64, typed=True)
def _flags(eps: float, interleaved) -> Optional[int]:
    """The plan's flags: interleaved and the bits of eps; None for values that are refused."""
    if not 0.0 <= eps < 1e30:
        return None
    return struct.unpack("I", struct.pack("f", eps))[0] << 1 | interleaved


def _validate(fn, q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved):
    import torch

    bf16, device = torch.bfloat16, getattr(q, "device", None)
    check_tensor(fn, "q", q, bf16, (None,) * 4, None)
    b, h, s, d = q.shape
    need(fn, d in (64, 128), f"the head size must be 64 or 128, got {d}")
    check_tensor(fn, "k", k, bf16, (b, None, s, d), device)
    check_tensor(fn, "q_weight", q_weight, (bf16, torch.float32), (d,), device)
    check_tensor(fn, "k_weight", k_weight, q_weight.dtype, (d,), device)
    check_tensor(fn, "cos", cos, torch.float32, (None, d // 2), device)
    check_tensor(fn, "sin", sin, torch.float32, (cos.shape[0], d // 2), device)
    need(fn, 0 < cos.shape[0] <= INT_MAX, "the table has no rows")
    if positions is not None:
        ints = (torch.int32, torch.int64)
        if getattr(positions, "dim", lambda: 2)() == 1:
            check_tensor(fn, "positions", positions, ints, (s,), device, rows=False)
        else:
            check_tensor(fn, "positions", positions, ints, (b, s), device, rows=False)
    if not isinstance(eps, (int, float)) or not 0.0 <= eps < 1e30:
        raise ValueError(f"{fn}: eps must be a number >= 0, got {eps!r}")
    if not isinstance(interleaved, bool):
        raise TypeError(f"{fn}: interleaved must be a bool")
    need(fn, b * s * (h + k.shape[1]) < 1 << 29, "2^29 rows or more in one call")
    need(fn, b * -(-s * (h + k.shape[1]) * d // 4096) < 1 << 24, "2^24 workgroups or more in one call")
    return b, h, s, d, device


def _packed(q, k, q_out, k_out, dq, dk, q_weight, cos, sin, positions, eps):
    """The argument structure without its pointers."""
    import torch

    def side(x, g, out):
        b, h, s, _ = x.stride()
        gb, gh, gs = g.stride()[:3] if g is not None else (0, 0, 0)
        return _Side(None, None, None, None, b, h, s, gb, gh, gs, *out.stride()[:3], x.shape[1], 0)

    pb = ps = 0
    if positions is not None:
        pb, ps = (0, positions.stride(0)) if positions.dim() == 1 else positions.stride()
    flags = (1 if q_weight.dtype == torch.float32 else 0) | (
        2 if positions is not None and positions.dtype == torch.int64 else 0)
    return _Args(side(q, dq, q_out), side(k, dk, k_out), None, None, None, None, pb, ps, cos.stride(0), sin.stride(0),
                 q.shape[0], q.shape[2], cos.shape[0], flags, eps)


# what a given output and another tensor of the call must not share, with the pairs that may be one tensor last
_FORWARD_PAIRS = ("q_out", "k_out", "q_out", "k", "k_out", "q", "q_out", "q", "k_out", "k")
_BACKWARD_PAIRS = ("dq", "dk", "dq", "dk_out", "dq", "k", "dk", "dq_out", "dk", "q", "dq_weight", "dk_weight",
                   "dq", "dq_out", "dq", "q", "dk", "dk_out", "dk", "k")


def qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions=None, eps: float = 1e-6, interleaved: bool = False,
                 q_out=None, k_out=None) -> Tuple[object, object]:
    """The RMS norm of every head of ``q`` ``[B, H, S, D]`` and ``k`` ``[B, H_kv, S, D]``
    (bf16, D = 64 or 128; views of a fused projection are read as they lie),
    scaled by ``q_weight`` / ``k_weight`` (``[D]``, bf16 or fp32), and the rotation
    by the token's position, in one launch; returns ``(q_out, k_out)``, bf16.

    ``cos`` and ``sin`` are ``[positions, D / 2]`` fp32 (``rope_table``).  The
    rotation turns pairs ``(i, i + D / 2)``, or ``(2 i, 2 i + 1)`` with
    ``interleaved``.  ``positions`` is int32 or int64, ``[S]`` or ``[B, S]`` (default
    ``0 .. S - 1``); the rows of a position outside the table become NaN.
    ``q_out`` may be ``q`` itself and ``k_out`` ``k``; memory that an output shares
    otherwise with the other, ``q`` or ``k`` is refused."""
    import torch

    fn = "qk_norm_rope"
    flags, done = _flags(eps, interleaved) if type(eps) is float and type(interleaved) is bool else None, None
    given = None
    if q_out is not None or k_out is not None:
        need(fn, q_out is not k_out, "q_out and k_out are one tensor")
        apart(fn, _FORWARD_PAIRS, 3, q_out, k_out, q_out, k, k_out, q, q_out, q, k_out, k)
        given = q_out, k_out
        q_out, k_out = own(q_out, q), own(k_out, k)
    if k_weight is q_weight:
        k_weight = own(k_weight, q_weight)
    if flags is not None:
        done = _forward_plans.run(flags, q, k, q_weight, k_weight, cos, sin, positions, q_out, k_out)
        if done is not None and done is not False:
            return _results(given, done)
    b, h, s, d, device = _validate(fn, q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)
    rec = _forward_plans.recording(done, q, k, q_weight, k_weight, cos, sin, positions, q_out, k_out)
    q_out = _output(fn, "q_out", q_out, q, rec)
    k_out = _output(fn, "k_out", k_out, k, rec)
    if b * s * (h + k.shape[1]) == 0:
        return _results(given, (q_out, k_out))
    args = _packed(q, k, q_out, k_out, None, None, q_weight, cos, sin, positions, eps)
    rows = 4096 // d   # rows of a workgroup, all of one sequence
    launch(rec, device, "qk_norm_rope.hsaco", f"wir_qk_norm_rope_d{d}" + ("_inter" if interleaved else ""),
           (b * -(-s * (h + k.shape[1]) // rows), 1, 1), (256, 1, 1), args,
           {"q.x": q, "q.out": q_out, "q.w": q_weight, "k.x": k, "k.out": k_out, "k.w": k_weight, "cos": cos,
            "sin": sin, "pos": positions})
    if rec:
        _forward_plans.add(flags, rec, q_out, k_out)
    return _results(given, (q_out, k_out))


def _results(given, done):
    """The tensors that the caller gave, where it did."""
    return done if given is None else tuple(x if g is None else g for g, x in zip(given, done))


def _output(fn, name, out, like, rec):
    import torch

    if out is None:
        return rec.alloc(torch.empty(like.shape, dtype=like.dtype, device=like.device))
    check_tensor(fn, name, out, like.dtype, like.shape, like.device)
    check_written(fn, name, out)
    return out


def qk_norm_rope_backward(dq_out, dk_out, q, k, q_weight, k_weight, cos, sin, positions=None, eps: float = 1e-6,
                          interleaved: bool = False, dq=None, dk=None, dq_weight=None, dk_weight=None,
                          workspace=None):
    """Gradients ``(dq, dk, dq_weight, dk_weight)`` of ``qk_norm_rope`` from
    those of its outputs (``dq_out``, ``dk_out``, bf16, shaped as ``q`` and ``k``, any
    row-aligned layout) and its inputs; ``dq`` and ``dk`` are bf16, the weights'
    gradients fp32 sums over all rows, added in an order that the shapes fix.
    ``dq`` may be ``dq_out`` or ``q`` itself and ``dk`` ``dk_out`` or ``k``; memory that
    they share otherwise with one another or with those is refused.
    ``workspace`` holds the workgroups' partial sums (fp32, at least
    ``1025 * D`` elements, allocated if omitted); one call at a time may use it."""
    import torch

    fn = "qk_norm_rope_backward"
    flags, done = _flags(eps, interleaved) if type(eps) is float and type(interleaved) is bool else None, None
    given = None
    if dq is not None or dk is not None or dq_weight is not None or dk_weight is not None:
        need(fn, dq is None or dq is not dk, "dq and dk are one tensor")
        need(fn, dq_weight is None or dq_weight is not dk_weight, "dq_weight and dk_weight are one tensor")
        apart(fn, _BACKWARD_PAIRS, 6, dq, dk, dq, dk_out, dq, k, dk, dq_out, dk, q, dq_weight, dk_weight,
              dq, dq_out, dq, q, dk, dk_out, dk, k)
        given = dq, dk, dq_weight, dk_weight
        dq, dk = own(own(dq, dq_out), q), own(own(dk, dk_out), k)
    if k_weight is q_weight:
        k_weight = own(k_weight, q_weight)
    tensors = (dq_out, dk_out, q, k, q_weight, k_weight, cos, sin, positions, dq, dk, dq_weight, dk_weight)
    if flags is not None and workspace is None:
        done = _backward_plans.run(flags, *tensors)
        if done is not None and done is not False:
            return _results(given, done)
    b, h, s, d, device = _validate(fn, q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)
    check_tensor(fn, "dq_out", dq_out, q.dtype, q.shape, device)
    check_tensor(fn, "dk_out", dk_out, k.dtype, k.shape, device)
    rec = _backward_plans.recording(done, *tensors)
    dq = _output(fn, "dq", dq, q, rec)
    dk = _output(fn, "dk", dk, k, rec)
    weights = []
    for name, w in (("dq_weight", dq_weight), ("dk_weight", dk_weight)):
        if w is None:
            w = rec.alloc(torch.empty(d, dtype=torch.float32, device=device))
        check_tensor(fn, name, w, torch.float32, (d,), device)
        weights.append(w)
    hk = k.shape[1]
    if b * s * (h + hk) == 0:
        for w in weights:
            w.zero_()
        return _results(given, (dq, dk, *weights))
    args = _packed(q, k, dq, dk, dq_out, dk_out, q_weight, cos, sin, positions, eps)
    args.q.blocks, args.k.blocks = _blocks(b * s * h, b * s * hk, d)
    floats = (args.q.blocks + args.k.blocks) * d
    if workspace is None:
        workspace = rec.alloc(torch.empty(floats, dtype=torch.float32, device=device))
    check_tensor(fn, "workspace", workspace, torch.float32, (None,), device)
    need(fn, workspace.numel() >= floats, f"workspace needs {floats} elements")
    launch(rec, device, "qk_norm_rope.hsaco", f"wir_qk_norm_rope_bwd_d{d}" + ("_inter" if interleaved else ""),
           (args.q.blocks + args.k.blocks, 1, 1), (256, 1, 1), args,
           {"q.x": q, "q.g": dq_out, "q.out": dq, "q.w": q_weight, "k.x": k, "k.g": dk_out, "k.out": dk,
            "k.w": k_weight, "cos": cos, "sin": sin, "pos": positions, "partial": workspace})
    launch(rec, device, "qk_norm_rope.hsaco", "wir_rope_weight_grad", (d // 32, 2, 1), (256, 1, 1),
           _GradArgs(None, None, None, args.q.blocks, args.k.blocks, d),
           {"partial": workspace, "q": weights[0], "k": weights[1]})
    if rec:
        _backward_plans.add(flags, rec, dq, dk, *weights)
    return _results(given, (dq, dk, *weights))


def _blocks(q_rows: int, k_rows: int, d: int) -> Tuple[int, int]:
    """Workgroups of the backward for the rows of q and of k: one for each
    ``4096 / d`` rows, up to 1024 (four on each of 256 CUs) in the rows' ratio."""
    most = 1024
    each = [-(-n * d // 4096) for n in (q_rows, k_rows)]
    if sum(each) > most:
        qb = min(max(round(most * q_rows / (q_rows + k_rows)), 1 if q_rows else 0), most - (1 if k_rows else 0))
        each = [min(qb, each[0]), min(most - qb, each[1])]
    return each[0], each[1]


__all__ = ["rope_table", "qk_norm_rope", "qk_norm_rope_backward"]
