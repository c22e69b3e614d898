"""What the public calls over hand-written kernels share: argument checks and
launches that are right on any device and leave a launch plan."""
from __future__ import annotations

import contextlib
import ctypes
import functools
from typing import Dict, Optional, Sequence

from warpir_amd import plans
from warpir_amd.plans import Plans
from warpir_amd.runtime import RawKernel, check

INT_MAX = 2 ** 31 - 1


def need(fn: str, ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(f"{fn}: {what}")


def check_tensor(fn: str, name: str, t, dtypes, shape: Sequence[int], device, rows: bool = True) -> None:
    """Refuse a tensor that the kernels cannot address: its type, dtype, shape
    and device, and for ``rows`` the last dimension's stride and the 16-byte
    alignment of its rows.  ``shape`` entries of None match anything."""
    import torch

    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{fn}: {name} must be a torch.Tensor")
    dtypes = dtypes if isinstance(dtypes, tuple) else (dtypes,)
    if t.dtype not in dtypes:
        raise TypeError(f"{fn}: {name} must be {' or '.join(str(d).replace('torch.', '') for d in dtypes)}, "
                        f"got {t.dtype}")
    if t.dim() != len(shape) or any(w is not None and w != g for w, g in zip(shape, t.shape)):
        want = ", ".join("*" if w is None else str(w) for w in shape)
        raise ValueError(f"{fn}: {name} must have shape [{want}], got {list(t.shape)}")
    if not t.is_cuda:
        raise ValueError(f"{fn}: {name} must be a GPU tensor")
    if device is not None and t.device != device:
        raise ValueError(f"{fn}: all tensors must be on one device")
    if t.numel() == 0:
        return
    if rows:
        size = t.element_size()
        if t.shape[-1] > 1 and t.stride(-1) != 1:
            raise ValueError(f"{fn}: {name}'s last dimension must be contiguous")
        if t.data_ptr() % 16 or any(n > 1 and s * size % 16 for n, s in zip(t.shape[:-1], t.stride()[:-1])):
            raise ValueError(f"{fn}: {name}'s rows must be 16-byte aligned")
    if not t.data_ptr():   # a kernel would follow the null pointer
        raise ValueError(f"{fn}: {name} has no memory (a fake or meta tensor)")


def check_written(fn: str, name: str, t) -> None:
    """Refuse a destination in which two elements may share a place."""
    span = 1
    for size, stride in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n > 1), key=lambda x: x[1]):
        if stride < span:
            raise ValueError(f"{fn}: {name}'s elements overlap (a broadcast tensor cannot be written)")
        span = stride * (size - 1) + span


def apart(fn: str, names: Sequence[str], strict: int, *tensors) -> None:
    """Refuse pairs of ``tensors`` (named by ``names``) that have memory in common:
    a kernel's workgroups write one while others read or write the other.  Past
    the first ``strict`` pairs one layout at one address is no such pair: a row is
    read and written by the same lanes.  None has no memory."""
    mod = plans._native
    if mod is None:
        import torch

        if not torch.cuda.is_available():
            return   # (nothing runs)
        mod = plans.native()
    first = mod.meets(strict, *tensors)
    if first >= 0:
        raise ValueError(f"{fn}: {names[2 * first]} and {names[2 * first + 1]} have memory in common")


def own(t, other):
    """``t`` as a tensor of its own where it is ``other``: a call that gives one
    tensor twice has no plan."""
    return t.view_as(t) if t is other and hasattr(t, "view_as") else t


@functools.lru_cache(maxsize=None)
def _kernel(filename: str, symbol: str, device: int) -> RawKernel:
    return RawKernel(filename, symbol)   # (a code object is loaded for one device)


def on(device):
    """The tensors' device as the current one, where it is another."""
    import torch

    if device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def launch(rec, device, filename: str, symbol: str, grid, block, args: ctypes.Structure,
           tensors: Dict[str, object], offsets: Optional[Dict[str, int]] = None) -> None:
    """Launch a hand-written kernel on the current stream of *device* and note
    it for a plan.  ``tensors`` names the pointer fields of *args* ("q.x" is
    field x of field q); ``offsets`` the bytes past a tensor's data."""
    import torch

    pointers = []
    for path, t in tensors.items():
        if t is None:
            continue
        part, base, typ = args, 0, type(args)
        *outer, last = path.split(".")
        for f in outer:
            base += getattr(typ, f).offset
            part = getattr(part, f)
            typ = type(part)
        off = offsets.get(path, 0) if offsets else 0
        setattr(part, last, t.data_ptr() + off)
        if rec:
            pointers.append((base + getattr(typ, last).offset, rec.slot(t), off))
    kernel = _kernel(filename, symbol, device.index)
    with on(device):
        kernel.launch(grid, block, args, stream=torch.cuda.current_stream(device).cuda_stream)
    if rec:
        rec.raw(kernel._function, grid, block, args, pointers)


class DevicePlans(Plans):
    """Plans that are replayed on the current device only: the default stream
    of another one has no handle of its own."""

    _one_device = False

    def run(self, flags: int, *tensors):
        if self._one_device:   # (the common call: no more Python than this)
            r = plans._native.run(self._table, flags, *tensors)
            if type(r) is not int:
                return r
            check(r, self.what)
        import torch

        first = tensors[0]
        if not getattr(first, "is_cuda", False) or first.device.index != torch.cuda.current_device():
            return None
        r = super().run(flags, *tensors)
        self._one_device = self._table is not None and torch.cuda.device_count() == 1
        return r


__all__ = ["apart", "check_tensor", "check_written", "need", "own", "launch", "on", "DevicePlans", "INT_MAX"]
