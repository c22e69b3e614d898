"""Attention over packed sequences of different lengths and its gradients
(``csrc/attn_packed.hip``, ``csrc/attn_packed_bwd.hip``)."""
from __future__ import annotations

import ctypes
from typing import Tuple

from warpir_amd.handwritten import INT_MAX, DevicePlans, apart, check_tensor, check_written, launch, need, own

_forward_plans = DevicePlans("attention_packed")
_backward_plans = DevicePlans("attention_packed_backward")

ROWS = 128   # query rows, or keys, of a workgroup (csrc/wir_packed.h)


class _Args(ctypes.Structure):
    _fields_ = [*((n, ctypes.c_void_p) for n in ("q", "k", "v", "out", "lse", "offsets")),
                *((n, ctypes.c_longlong) for n in ("qh", "qt", "kh", "kt", "vh", "vt", "oh", "ot", "lh", "lt")),
                *((n, ctypes.c_int) for n in ("batch", "tokens", "heads", "group", "blocks", "flags"))]


class _GradArgs(ctypes.Structure):
    _fields_ = [*((n, ctypes.c_void_p) for n in ("q", "k", "v", "o", "d_o", "lse", "offsets", "dq", "dk", "dv", "stats")),
                *((n, ctypes.c_longlong) for n in ("qh", "qt", "kh", "kt", "vh", "vt", "oh", "ot", "gh", "gt", "lh", "lt",
                                                   "dqh", "dqt", "dkh", "dkt", "dvh", "dvt")),
                *((n, ctypes.c_int) for n in ("batch", "tokens", "heads", "group", "blocks", "flags"))]


def _validate(fn, q, k, v, offsets, causal):
    """(heads, key/value heads, tokens, D, batch, device)"""
    import torch

    bf16, device = torch.bfloat16, getattr(q, "device", None)
    check_tensor(fn, "q", q, bf16, (None,) * 3, None)
    heads, tokens, d = q.shape
    need(fn, d in (64, 128), f"the head size must be 64 or 128, got {d}")
    check_tensor(fn, "k", k, bf16, (None, tokens, d), device)
    check_tensor(fn, "v", v, bf16, k.shape, device)
    shared = k.shape[0]
    need(fn, shared > 0 and heads > 0 and heads % shared == 0,
         f"{heads} query heads are not a multiple of {shared} key/value heads")
    check_tensor(fn, "offsets", offsets, torch.int32, (None,), device, rows=False)
    batch = offsets.shape[0] - 1
    need(fn, batch >= 0, "offsets must hold the end of each sequence behind a first 0")
    need(fn, batch == 0 or offsets.stride(0) == 1, "offsets must be contiguous")
    if not isinstance(causal, bool):
        raise TypeError(f"{fn}: causal must be a bool")
    need(fn, tokens + batch <= INT_MAX - 2 * ROWS, "2^31 tokens or more in one call")
    for name, x in (("q", q), ("k", k), ("v", v)):
        need(fn, tokens < 2 or x.stride(1) < 1 << 23, f"{name}'s tokens are 2^23 elements or more apart")
    need(fn, (tokens // ROWS + batch + 1) * heads < 1 << 23, "2^32 threads or more in one call")
    return heads, shared, tokens, d, batch, device


def _by_token(heads, tokens, d, device, rec):
    """[H, T, D], a token's heads next to one another: as a projection reads it."""
    import torch

    return rec.alloc(torch.empty(tokens, heads, d, dtype=torch.bfloat16, device=device).transpose(0, 1))


# what a given result and another tensor of the call must not share; past the first ones, pairs that may be one tensor
_FORWARD_PAIRS = ("out", "lse", "out", "k", "out", "v", "out", "offsets", "lse", "q", "lse", "k", "lse", "v", "lse", "offsets",
                  "out", "q")


def attention_packed(q, k, v, offsets, causal: bool = True, out=None, lse=None) -> Tuple[object, object]:
    """Attention over packed sequences: ``q`` ``[H, T, D]``, ``k`` and ``v`` ``[H_kv, T, D]``
    (bf16, D = 64 or 128, H a multiple of H_kv; any 16-byte aligned rows, so
    views of a fused projection are read as they lie).  Returns ``(O, LSE)``,
    bf16 ``[H, T, D]`` and fp32 ``[H, T]`` (natural log) as ``api.attention_forward``.

    Sequence ``i`` is tokens ``offsets[i] .. offsets[i + 1] - 1`` (int32, ascending from
    0, on the GPU; sequences may be empty); its tokens see one another, with
    ``causal`` only those up to their own.  Tokens behind ``offsets[-1]`` belong to no
    sequence: a given ``out`` or ``lse`` keeps what it has there, an allocated one
    holds 0 and -inf.  In a captured graph the offsets may change between
    replays.  What a row does not see does not reach it, be it infinite or NaN.  A key
    whose score is -inf weighs nothing; a row with no other has O NaN and LSE -inf.
    Sums over the keys are divided by their weight at the end: values of v up to 2^96
    in magnitude cannot overflow on the way.

    An allocated ``O`` lies token by token, so that ``O.transpose(0, 1).reshape(T, H * D)``
    is the next product's operand as it is.  ``out`` may be ``q`` itself; other memory
    that ``out`` or ``lse`` shares with a tensor of the call is refused."""
    import torch

    fn, done, given = "attention_packed", None, None
    if out is not None or lse is not None:
        apart(fn, _FORWARD_PAIRS, 8, out, lse, out, k, out, v, out, offsets, lse, q, lse, k, lse, v, lse, offsets, out, q)
        given = out, lse
        out = own(out, q)
    planned = type(causal) is bool
    if planned:
        done = _forward_plans.run(causal, q, k, v, offsets, out, lse)
        if done is not None and done is not False:
            return _results(given, done)
    heads, shared, tokens, d, batch, device = _validate(fn, q, k, v, offsets, causal)
    rec = _forward_plans.recording(done, q, k, v, offsets, out, lse)
    flags = (1 if out is None else 0) | (2 if lse is None else 0)
    if out is not None:
        check_tensor(fn, "out", out, torch.bfloat16, q.shape, device)
        check_written(fn, "out", out)
    if lse is not None:
        check_tensor(fn, "lse", lse, torch.float32, q.shape[:2], device, rows=False)
        check_written(fn, "lse", lse)
    if out is None:
        out = _by_token(heads, tokens, d, device, rec)
    if lse is None:
        lse = rec.alloc(torch.empty(heads, tokens, dtype=torch.float32, device=device))
    if tokens == 0:
        return _results(given, (out, lse))
    kind, rows, waves, two = _forward_form(heads, shared, tokens, batch, d)
    blocks = tokens // rows + batch + 1
    args = _Args(*[None] * 6, *(s for x in (q, k, v, out) for s in x.stride()[:2]), *lse.stride(), batch, tokens, heads,
                 heads // shared, blocks, flags | (4 if two else 0))
    launch(rec, device, "attn_packed_split.hsaco" if kind == "_split" else "attn_packed.hsaco", f"wir_attn_packed_d{d}{kind}" + ("_causal" if causal else ""),
           (blocks * (heads // 2 if two else heads), 1, 1), (64 * waves, 1, 1), args,
           {"q": q, "k": k, "v": v, "out": out, "lse": lse, "offsets": offsets})
    if rec:
        _forward_plans.add(causal, rec, out, lse)
    return _results(given, (out, lse))


# A launch of the split kernels (32 rows a workgroup, whose waves divide the other side) against one of 128 rows: us of
# 64 keys (queries) that a workgroup of 128 rows walks, of the start of one of 32, and its part of that walk.  By launches of
# 5 x 90 to 2 x 4096 tokens, 8/8 and 16/4 heads, causal; us, 128 rows / 32: forward D = 64, 8 heads, 1 x 512 11.2 / 7.4, 2 x
# 1024 16.8 / 14.2, 8 x 256 8.5 / 10.5; dQ D = 128 1 x 512 19.0 / 13.0, 1 x 4096 106 / 113, 32 x 64 13.6 / 22.4; dK/dV D = 64, 16/4
# heads, 1 x 512 44.9 / 18.2, 8 x 512 46.0 / 33.0, 64 x 64 14.9 / 21.0, D = 128 2 x 1024 108 / 63, 8 x 1024 117 / 155.  The
# rule's choice is within 0.7% (geometric mean) of the faster one, dQ's at D = 64 and dK/dV's at 128 included.
_SPLIT_US = {("forward", 64): (0.72, 2.67, 0.22), ("forward", 128): (1.23, 3.18, 0.27), ("dq", 64): (1.19, 3.55, 0.18),
             ("dq", 128): (1.91, 4.64, 0.19), ("dkdv", 64): (1.29, 3.70, 0.17), ("dkdv", 128): (1.96, 4.26, 0.26)}


def _splits(part: str, heads: int, walks: int, tokens: int, batch: int, d: int) -> bool:
    """Whether a launch over ``heads`` heads, whose workgroups walk a sequence ``walks``
    times, goes to the split kernels.  The lengths are on the GPU: their average decides."""
    tile, start, share = _SPLIT_US[part, d]
    walk = tile * walks * tokens / (64 * max(batch, 1))
    rounds = (tokens / 32 + batch) * heads / 256   # of one workgroup a CU
    rounds = 1 if rounds <= 1 else rounds + 0.5
    return 3 + rounds * (start + share * walk) < 5.5 + walk


def _forward_form(heads: int, shared: int, tokens: int, batch: int, d: int) -> Tuple[str, int, int, bool]:
    """(kind of the kernel, query rows and waves of a workgroup, whether it takes two heads) of the forward.

    Eight waves are two groups of four with the same tiles: two heads that share
    keys and values, or 256 rows of one head.  They pay at D = 128 in long sequences;
    the lengths are on the GPU, so their average decides.  us, four / eight waves,
    batches of 32768 tokens in sequences of 128, 256, 512, 1024, 2048, 4096:
    32/8 heads, not causal 290 / 327, 240 / 257, 359 / 334, 558 / 532, 976 / 949, 1840
    / 1750; causal 284 / 338, 208 / 225, 260 / 263, 368 / 371, 589 / 587, 1024 / 992;
    16/16 heads, not causal 170 / 157, 139 / 213, 192 / 200, 283 / 285, 506 / 494, 932 / 893."""
    if _splits("forward", heads, 1, tokens, batch, d):
        return "_split", 32, 4, False
    average = tokens / max(batch, 1)
    two = heads // shared % 2 == 0
    if d == 128 and average >= (512 if two else 2048) and tokens * heads >= 1 << 17:   # (two such workgroups a CU)
        return "_w8", 128 if two else 256, 8, two
    return "", 128, 4, False


def _results(given, done):
    """The tensors that the caller gave, where it did."""
    return done if given is None else tuple(x if g is None else g for g, x in zip(given, done))


# the same of a given gradient or workspace
_BACKWARD_PAIRS = ("dq", "dk", "dq", "dv", "dk", "dv", "dq", "q", "dq", "k", "dq", "v", "dq", "o", "dq", "do", "dq", "lse", "dq", "offsets",
                   "dk", "q", "dk", "v", "dk", "o", "dk", "do", "dk", "lse", "dk", "offsets",
                   "dv", "q", "dv", "k", "dv", "o", "dv", "do", "dv", "lse", "dv", "offsets",
                   "workspace", "q", "workspace", "k", "workspace", "v", "workspace", "o", "workspace", "do", "workspace", "lse",
                   "workspace", "offsets", "workspace", "dq", "workspace", "dk", "workspace", "dv", "dk", "k", "dv", "v")


def attention_packed_backward(q, k, v, o, lse, do, offsets, causal: bool = True, dq=None, dk=None, dv=None,
                              workspace=None) -> Tuple[object, object, object]:
    """Gradients ``(dq, dk, dv)`` (bf16) of ``attention_packed`` from its inputs, its
    outputs ``o`` and ``lse`` and the gradient ``do`` of ``o`` (bf16 ``[H, T, D]``, any
    row-aligned layout); ``causal`` as in the forward.  The sums over a
    key/value head's query heads are in 32 bits, in an order that the shapes and the
    lengths fix (T with the tokens behind the last sequence).

    Tokens behind ``offsets[-1]`` get no gradient: given tensors keep what they
    have there, allocated ones (which lie token by token) hold 0.  ``dk`` may be
    ``k`` itself and ``dv`` ``v``; other memory that they or ``workspace`` share with a
    tensor of the call is refused.  ``workspace`` holds two numbers for each query head
    and token (fp32, at least ``2 * H * T`` elements, allocated if omitted); one call at
    a time may use it."""
    import torch

    fn, done, given = "attention_packed_backward", None, None
    if dq is not None or dk is not None or dv is not None or workspace is not None:
        ws = workspace
        apart(fn, _BACKWARD_PAIRS, 32, dq, dk, dq, dv, dk, dv, dq, q, dq, k, dq, v, dq, o, dq, do, dq, lse, dq, offsets,
              dk, q, dk, v, dk, o, dk, do, dk, lse, dk, offsets, dv, q, dv, k, dv, o, dv, do, dv, lse, dv, offsets,
              ws, q, ws, k, ws, v, ws, o, ws, do, ws, lse, ws, offsets, ws, dq, ws, dk, ws, dv, dk, k, dv, v)
        given = dq, dk, dv
        dk, dv = own(dk, k), own(dv, v)
    tensors = (q, k, v, o, lse, do, offsets, dq, dk, dv)
    if type(causal) is bool and workspace is None:
        done = _backward_plans.run(causal, *tensors)
        if done is not None and done is not False:
            return _results(given, done)
    heads, shared, tokens, d, batch, device = _validate(fn, q, k, v, offsets, causal)
    for name, x in (("o", o), ("do", do)):
        check_tensor(fn, name, x, torch.bfloat16, q.shape, device)
    need(fn, tokens < 2 or do.stride(1) < 1 << 23, "do's tokens are 2^23 elements or more apart")
    check_tensor(fn, "lse", lse, torch.float32, q.shape[:2], device, rows=False)
    floats, flags = 2 * heads * tokens, 0
    for name, x, like in (("dq", dq, q), ("dk", dk, k), ("dv", dv, v)):
        if x is not None:
            check_tensor(fn, name, x, torch.bfloat16, like.shape, device)
            check_written(fn, name, x)
    if workspace is not None:
        check_tensor(fn, "workspace", workspace, torch.float32, (None,), device)
        need(fn, workspace.numel() >= floats, f"workspace needs {floats} elements")
    rec = _backward_plans.recording(done, *tensors)
    grads = [dq, dk, dv]
    for i, like in enumerate((q, k, v)):
        if grads[i] is None:
            flags |= 1 << i
            grads[i] = _by_token(like.shape[0], tokens, d, device, rec)
    if workspace is None:
        workspace = rec.alloc(torch.empty(floats, dtype=torch.float32, device=device))
    if tokens == 0:
        return _results(given, tuple(grads))
    names = {"q": q, "k": k, "v": v, "o": o, "d_o": do, "lse": lse, "offsets": offsets, "dq": grads[0], "dk": grads[1],
             "dv": grads[2], "stats": workspace}
    strides = [s for x in (q, k, v, o, do, lse, *grads) for s in x.stride()[:2]]
    for part, programs in (("dq", heads), ("dkdv", shared)):
        split = _splits(part, programs, heads // programs, tokens, batch, d)
        blocks = tokens // (32 if split else ROWS) + batch + 1
        threads = 512 if part == "dkdv" and (d == 64) == split else 256
        args = _GradArgs(*[None] * 11, *strides, batch, tokens, heads, heads // shared, blocks, flags)
        launch(rec, device, "attn_packed_split.hsaco" if split else "attn_packed_bwd.hsaco",
               f"wir_attn_packed_{part}_d{d}" + ("_split" if split else "") + ("_causal" if causal else ""),
               (blocks * programs, 1, 1), (threads, 1, 1), args, names)
    if rec:
        _backward_plans.add(causal, rec, *grads)
    return _results(given, tuple(grads))


__all__ = ["attention_packed", "attention_packed_backward"]
