"""What the row operators (layer norm, log probabilities, 8-bit kept
activations) share: element type codes of the C ABI, the view of a tensor as
rows, argument checks and the device guard around a launch."""

from __future__ import annotations

import contextlib
from typing import Tuple

import torch

from zookeeper_amd.ops import _native

# element type codes of the C ABI (csrc/kernels/rows.h)
DTYPE_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_FLOATS = (torch.float32, torch.bfloat16, torch.float16, torch.float64)

# Raw hipStream_t of torch's current stream on a device index.
raw_stream = torch._C._cuda_getCurrentRawStream

_HERE = contextlib.nullcontext()


def call(fn, what: str, *args) -> None:
    """A native launch and its error check."""
    rc = fn(*args)
    if rc or _native._DEBUG_SYNC:
        _native.check(rc, what)


def use_kernels(t: torch.Tensor, what: str) -> bool:
    """True for a GPU tensor (the HIP kernels run; :func:`_native.lib` raises
    if the library is missing), False for the plain PyTorch form: host tensors,
    or the native path switched off with ``ZK_NATIVE=0``."""
    if t.is_cuda and t.dtype in DTYPE_CODES and _native.available():
        return True
    if not t.is_cuda or _native.native_disabled():
        if not t.is_floating_point():
            raise ValueError(f"{what}: expected a floating-point tensor, got {t.dtype}")
        return False
    if t.dtype not in DTYPE_CODES:
        raise ValueError(f"{what}: expected float32, bfloat16 or float16, got {t.dtype}")
    return True


def guard(t: torch.Tensor):
    """Context that makes ``t``'s device the current one for a launch."""
    if t.device.index == torch._C._cuda_getDevice():
        return _HERE
    return torch.cuda.device(t.device)


def rows_of(t: torch.Tensor) -> Tuple[torch.Tensor, int, int]:
    """``(t2, rows, row stride)``: ``t`` as rows of its last dimension with unit
    stride inside a row -- a view where the strides allow it (padded, sliced or
    broadcast rows), a contiguous copy otherwise."""
    cols = t.shape[-1]
    if t.is_contiguous():
        return t, t.numel() // cols if cols else 0, cols
    if t.dim() != 2:
        t = t.reshape(-1, cols)
    if cols > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t, t.shape[0], t.stride(0)


def check_param(p, cols: int, x: torch.Tensor, what: str) -> None:
    if p.shape == (cols,) and p.device == x.device and p.dtype in _FLOATS:
        return
    if p.dim() != 1 or p.shape[0] != cols:
        raise ValueError(f"{what}: expected shape ({cols},), got {tuple(p.shape)}")
    if p.device != x.device:
        raise ValueError(f"{what}: on {p.device}, the input is on {x.device}")
    if not p.is_floating_point():
        raise ValueError(f"{what}: expected a floating-point tensor, got {p.dtype}")


def as_fp32(p):
    """A parameter as the kernels read it: fp32, contiguous (None stays None)."""
    if p is None or (p.dtype == torch.float32 and p.is_contiguous()):
        return p
    return p.detach().to(torch.float32).contiguous()


def ptr(t):
    return None if t is None else t.data_ptr()


def refuse_twice(what: str) -> None:
    """Raised by a backward that runs with gradients recorded, which is what
    ``create_graph=True`` does: the kernels' gradients are not differentiable
    themselves and would count as constants."""
    raise RuntimeError(f"{what}: the gradient is not differentiable (create_graph=True)")
