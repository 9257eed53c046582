"""What the row operators (layer norm, log probabilities, 8-bit kept
activations) share: element type codes of the C ABI, the view of a tensor as
rows, argument checks, the device guard around a launch and the writes into
flat gradient buffers."""

from __future__ import annotations

import contextlib
import weakref
from typing import Dict, Optional, Tuple

import torch
from torch.autograd import forward_ad

from zookeeper_amd.ops import _native

# element type codes of the C ABI (csrc/kernels/rows.h)
DTYPE_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_FLOATS = (torch.float32, torch.bfloat16, torch.float16, torch.float64)

# Raw hipStream_t of torch's current stream on a device index (a torch without GPU
# support lacks the name, and has no GPU tensors to need it).
raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)

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


def tracked() -> bool:
    """True while torch follows calls by other means than ``requires_grad``: tracing
    records an autograd function as one call, and forward-mode differentiation
    is refused by it.  A bare launch would be invisible to both."""
    return forward_ad._current_level >= 0 or torch._C._is_tracing()


def refuse_tracing(what: str) -> None:
    if torch._C._is_tracing():
        raise RuntimeError(f"{what}: cannot be traced (it is no autograd function)")


def guard(t: torch.Tensor):
    """Context that makes ``t``'s device the current one for a launch."""
    if t.device.index == torch._C._cuda_getDevice():
        return _HERE
    return torch.cuda.device(t.device)


def rows_of(t: torch.Tensor) -> Tuple[torch.Tensor, int, int]:
    """``(t2, rows, row stride)``: ``t`` as rows of its last dimension with unit
    stride inside a row -- a view where the strides allow it (padded, sliced or
    broadcast rows), a contiguous copy otherwise.  ``int``: sizes are tensors
    while a call is traced."""
    cols = int(t.shape[-1])
    if t.is_contiguous():
        return t, int(t.numel()) // cols if cols else 0, cols
    if t.dim() != 2:
        t = t.reshape(-1, cols)
    if cols > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t, int(t.shape[0]), int(t.stride(0))


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


class _Use:
    """One recorded use of a parameter whose gradient is still to come."""

    __slots__ = ("param", "__weakref__")

    def __init__(self, param):
        self.param = param


# Recorded uses by parameter (a use holds its parameter, so an id means one while any is
# left).  Not kept on the parameter itself: a module is saved with its parameters'
# attributes.
_USES: Dict[int, "weakref.WeakSet[_Use]"] = {}


def note_uses(*params):
    """Forward: a token for each parameter a data-parallel bucketer waits for
    (None otherwise).  A token lives as long as the recorded graph, so a graph
    that is dropped without a backward leaves none behind."""
    tokens = []
    for p in params:
        token = None
        if p is not None and getattr(p, "_zk_grad_ready", None) is not None:
            token = _Use(p)
            _USES.setdefault(id(p), weakref.WeakSet()).add(token)
        tokens.append(token)
    return tokens


def last_use_ready(p, token) -> None:
    """Backward: tell the bucketer that ``p``'s gradient is complete, once no
    other recorded use of ``p`` is to come (a layer applied twice)."""
    if token is not None:
        uses = _USES.get(id(p), ())
        if uses:
            uses.discard(token)
        if uses:
            return
        _USES.pop(id(p), None)
    _native.grad_ready(p)


# Streams that added into flat gradients, by backward pass and parameter.
_WRITERS: Dict[int, Dict[int, Tuple[torch.device, int]]] = {}


def _stream(device: torch.device, raw: int):
    if raw == 0:
        return torch.cuda.default_stream(device)
    return torch.cuda.ExternalStream(raw, device)


def _join_writers(task: int) -> None:
    for device, raw in set(_WRITERS.pop(task, {}).values()):
        if raw != raw_stream(device.index):
            torch.cuda.current_stream(device).wait_stream(_stream(device, raw))


def flat_grad(p) -> Optional[torch.Tensor]:
    """:func:`_native.direct_grad` for a parameter that may be used on several
    streams in one backward pass.  Autograd orders the gradients it accumulates
    and knows nothing of these: each write waits for the one before it on
    another stream, and the caller's stream for all of them at the pass's end."""
    g = _native.direct_grad(p)
    if g is None:
        return None
    task = torch._C._current_graph_task_id()
    if task < 0:  # not inside a backward pass: one stream, the caller's
        return g
    writers = _WRITERS.get(task)
    if writers is None:
        writers = _WRITERS[task] = {}
        torch.autograd.Variable._execution_engine.queue_callback(lambda: _join_writers(task))
    here = (g.device, raw_stream(g.device.index))
    last = writers.get(id(p), here)
    writers[id(p)] = here
    if last != here:
        torch.cuda.current_stream(g.device).wait_stream(_stream(*last))
    return g


def refuse_twice(what: str) -> None:
    """Raised by a backward that runs with gradients recorded, which is what
    ``create_graph=True`` does: the kernels' gradients are not differentiable
    themselves and would count as constants."""
    raise RuntimeError(f"{what}: the gradient is not differentiable (create_graph=True)")
