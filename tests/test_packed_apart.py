"""Memory that a packed operator's destinations and workspaces share with
another tensor of the call: what other workgroups still read, or write too, is refused
by name.  On CPU tensors, which would be refused next for being none of the GPU's."""
import os

import pytest
import torch

from warpir_amd import api, plans
from warpir_amd.runtime import PKG_DIR

pytestmark = pytest.mark.skipif(not os.path.exists(os.path.join(PKG_DIR, "_wir_plans.so")), reason="not built")

f32, i32, i8, bf16 = torch.float32, torch.int32, torch.int8, torch.bfloat16
H, HK, T, D = 4, 2, 30, 64


def _as(t, dtype, *shape):
    """Memory of ``t`` from its first element on, as another tensor."""
    n = 1
    for s in shape:
        n *= s
    flat = t.view(-1).view(dtype) if t.is_contiguous() else t
    return flat[:n].view(shape)


def _refused(call, what, **a):
    plans.native()
    with pytest.raises(ValueError, match=f"{what} have memory in common"):
        call(**a)


def _passes(call, **a):
    plans.native()
    with pytest.raises(ValueError, match="must be a GPU tensor"):
        call(**a)


def _attend():
    return dict(q=torch.zeros(H, T, D, dtype=bf16), k=torch.zeros(HK, T, D, dtype=bf16), v=torch.zeros(HK, T, D, dtype=bf16),
                offsets=torch.zeros(1000, dtype=i32)[:3])


@pytest.mark.parametrize("name", ["q", "k", "v"])
def test_lse_over_an_input(name):
    a = _attend()
    _refused(api.attention_packed, f"lse and {name}", **a, lse=_as(a[name], f32, H, T))


def test_results_over_offsets():
    a, room = _attend(), torch.zeros(H * T * D, dtype=bf16)
    a["offsets"] = room.view(i32)[:3]
    _refused(api.attention_packed, "out and offsets", **a, out=room.view(H, T, D))
    _refused(api.attention_packed, "lse and offsets", **a, lse=_as(room, f32, H, T))
    _passes(api.attention_packed, **a, out=a["q"], lse=torch.zeros(H, T))


def _gradients():
    a = _attend()
    a.update(o=torch.zeros(H, T, D, dtype=bf16), lse=torch.zeros(H * T * D)[:H * T].view(H, T), do=torch.zeros(H, T, D, dtype=bf16))
    return a


@pytest.mark.parametrize("name", ["dq", "dk", "dv"])
def test_gradients_over_lse_and_offsets(name):
    shape = (H if name == "dq" else HK, T, D)
    a, room = _gradients(), torch.zeros(H * T * D, dtype=bf16)
    _refused(api.attention_packed_backward, f"{name} and lse", **{**a, "lse": _as(room, f32, H, T)}, **{name: _as(room, bf16, *shape)})
    _refused(api.attention_packed_backward, f"{name} and offsets", **{**a, "offsets": room.view(i32)[:3]},
             **{name: _as(room, bf16, *shape)})


@pytest.mark.parametrize("name", ["q", "k", "v", "o", "do", "lse", "offsets", "dq", "dk", "dv"])
def test_workspace(name):
    a, room = _gradients(), torch.zeros(H * T * D, dtype=f32)
    shape = {"lse": (H, T), "offsets": (3,), "k": (HK, T, D), "v": (HK, T, D), "dk": (HK, T, D), "dv": (HK, T, D)}.get(name, (H, T, D))
    a[name] = _as(room, f32 if name == "lse" else i32 if name == "offsets" else bf16, *shape)
    _refused(api.attention_packed_backward, f"workspace and {name}", **a, workspace=room[:2 * H * T])


def test_gradients_that_pass():
    a, ws = _gradients(), torch.zeros(2 * H * T)
    _passes(api.attention_packed_backward, **a, workspace=ws)
    _passes(api.attention_packed_backward, **a, workspace=ws, dq=torch.zeros_like(a["q"]), dk=a["k"], dv=a["v"])
    _refused(api.attention_packed_backward, "dk and dv", **a, dk=a["k"], dv=a["k"].view(a["k"].shape))


def test_quantize():
    x = torch.zeros(64, 64, dtype=bf16)
    _refused(api.quantize_int8, "scale and x", x=x, scale=_as(x, f32, 64))
    _refused(api.quantize_int8, "scale and x", x=x, codes=torch.zeros(64, 64, dtype=i8), scale=_as(x, f32, 64))
    _refused(api.quantize_int8, "codes and x", x=x, codes=_as(x, i8, 64, 64))
    codes = torch.zeros(64, 64, dtype=i8)
    _refused(api.quantize_int8, "codes and scale", x=x, codes=codes, scale=_as(codes, f32, 64))
    _passes(api.quantize_int8, x=x, codes=codes, scale=torch.zeros(64))


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("side", [0, 1])
@pytest.mark.parametrize("name", ["cos", "sin", "positions"])
def test_rotation(name, side, back):
    call = api.rope_axes_backward if back else api.rope_axes
    outs = ("dq", "dk") if back else ("q_out", "k_out")
    ins = ("dq_out", "dk_out") if back else ("q", "k")
    room = torch.zeros(2 * 4 * 8 * 64, dtype=bf16)
    a = {ins[0]: torch.zeros(2, 4, 8, 64, dtype=bf16), ins[1]: torch.zeros(2, 2, 8, 64, dtype=bf16), "cos": torch.zeros(16, 24),
         "sin": torch.zeros(16, 24), "positions": torch.zeros(3, 8, dtype=i32), "sections": (8, 8, 8)}
    given = {outs[side]: _as(room, bf16, 2, 2 if side else 4, 8, 64)}
    _passes(call, **a, **given)
    _passes(call, **a, **{outs[side]: a[ins[side]]})
    a[name] = _as(room, i32, 3, 8) if name == "positions" else _as(room, f32, 16, 24)
    _refused(call, f"{outs[side]} and {name}", **a, **given)
