"""What the row operators (layer norm, log probabilities, 8-bit kept
activations) share: element type codes of the C ABI, the view of a tensor as
rows, argument checks, the device guard around a launch and the writes into
flat gradient buffers."""

from __future__ import annotations

import contextlib
import weakref
from typing import Dict, Optional, Set, Tuple

import torch
from torch.autograd import forward_ad

from zookeeper_amd.ops import _native

# element type codes of the C ABI (csrc/kernels/rows.h)
DTYPE_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_FLOATS = (torch.float32, torch.bfloat16, torch.float16, torch.float64)

# Raw hipStream_t of torch's current stream on a device index (a torch without GPU
# support lacks the name, and has no GPU tensors to need it).
raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
# The backward pass that this thread runs, -1 for none.
_task = torch._C._current_graph_task_id
_is_tracing = torch._C._is_tracing

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
    return forward_ad._current_level >= 0 or _is_tracing()


def refuse_tracing(what: str) -> None:
    if _is_tracing():
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


# --- flat gradients ------------------------------------------------------------

class _Pass:
    """The flat gradients written in one backward pass: the stream of each
    parameter's last write, the parameters written by uses that were recorded inside
    of another pass, and the streams of failed passes before it.  Called at the pass's
    end by autograd's engine, which holds the only lasting reference to it; a pass that
    fails is not called, only dropped."""

    __slots__ = ("writers", "inner", "left", "captured", "__weakref__")

    def __init__(self, device: torch.device):
        # a captured pass runs at its replays: nothing to wait for, and to wait for its
        # stream would draw the waiting one into the capture
        self.captured = _capturing(device)
        self.left = set() if self.captured else _unjoined(device)
        self.writers: Dict[int, Tuple[torch.device, int]] = {}
        self.inner: Set[int] = set()

    def __call__(self):
        _wait_for(self.left.union(self.writers.values()))
        self.left = set()
        self.writers.clear()

    def __del__(self):
        if not self.captured:
            _FAILED.update(self.left, self.writers.values())


_PASSES: "weakref.WeakValueDictionary[int, _Pass]" = weakref.WeakValueDictionary()
# Streams of failed passes, whose writes nobody has waited for.
_FAILED: Set[Tuple[torch.device, int]] = set()


def _unjoined(device: torch.device) -> Set[Tuple[torch.device, int]]:
    """Streams on ``device`` with writes that no ended pass has joined.  (Passes that are
    still there may be failed ones that the engine has not let go of.)"""
    left = _FAILED.copy()
    for current in list(_PASSES.values()):
        if not current.captured:
            left.update(list(current.writers.values()))
    left = {w for w in left if w[0] == device}
    # (a capture starts behind a synchronization)
    return set() if left and _capturing(device) else left


def _capturing(device: torch.device) -> bool:
    return device.type == "cuda" and torch.cuda.is_current_stream_capturing()


def _wait_for(writers) -> None:
    for device, raw in writers:
        if raw != _raw(device):
            torch.cuda.current_stream(device).wait_stream(_stream(device, raw))


def join_writers(device: torch.device) -> None:
    """The current stream waits for the writes that failed passes have left behind:
    before the buffer is cleared."""
    _wait_for(_unjoined(device))
    _FAILED.difference_update([w for w in _FAILED.copy() if w[0] == device])


def _raw(device: torch.device) -> int:
    return raw_stream(device.index) if device.type == "cuda" else 0


def _stream(device: torch.device, raw: int):
    if raw == 0:
        return torch.cuda.default_stream(device)
    return torch.cuda.ExternalStream(raw, device)


def _accumulated(p) -> None:
    """Autograd's hook behind the last use of ``p`` in a backward pass, whichever
    uses that pass has: every write into its flat gradient is enqueued, each behind
    the one before, so the bucketer may have it from the last one's stream on."""
    current = _PASSES.get(_task())
    last = current.writers.get(id(p)) if current is not None else None
    if last is None or id(p) in current.inner:
        return
    if last[1] == _raw(last[0]):
        _native.grad_ready(p)
    else:
        with torch.cuda.stream(_stream(*last)):
            _native.grad_ready(p)


def in_backward() -> bool:
    """True inside a backward pass.  A use recorded there belongs to a pass of its own
    inside that one (reentrant checkpointing), and others may follow."""
    return _task() >= 0


def _asked(ctx, p) -> Optional[bool]:
    """Whether this backward pass accumulates ``p``'s gradient (True), has no use for
    it (False: ``torch.autograd.grad`` of other tensors, ``backward(inputs=...)``) or
    hands it to its caller (None: ``torch.autograd.grad`` of ``p``)."""
    for node, _ in ctx.next_functions:
        if node is not None and getattr(node, "variable", None) is p:
            try:
                return torch._C._will_engine_execute_node(node)
            except RuntimeError:  # a leaf of torch.autograd.grad
                return None
    return True


def flat_grad(ctx, p, inner: bool) -> Tuple[bool, Optional[torch.Tensor]]:
    """``(needed, buffer)``: whether this pass wants ``p``'s gradient, and the flat
    buffer to add it to (None: return it to autograd).

    :func:`_native.direct_grad` for a parameter that may be used several times in
    one backward pass, on several streams.  Autograd orders the gradients it
    accumulates and knows nothing of these: each write waits for the one before it
    on another stream, and the caller's stream for all of them at the pass's end.

    The data-parallel bucketer hears of ``p`` once autograd is through with its last
    use of the pass (:func:`_accumulated`); ``inner`` (a use recorded in a backward
    pass): not before the bucketer's own end, as only that knows that no further
    inner pass follows.  A write that comes too late all the same raises."""
    task = _task()
    if task >= 0 and getattr(p, "_zk_direct_grad", False):
        asked = _asked(ctx, p)
        if not asked:
            return asked is None, None
    g = _native.direct_grad(p)
    if g is None:
        return True, None
    ready = getattr(p, "_zk_grad_ready", None)
    if getattr(ready, "launched", False):
        raise RuntimeError(
            "a gradient is written after its all-reduce was launched: the layer is used outside "
            "and inside of a reentrant checkpoint, or twice before the bucketer's finish()")
    if task < 0:  # not inside a backward pass: one stream, the caller's
        return True, g
    current = _PASSES.get(task)
    if current is None:
        current = _PASSES[task] = _Pass(g.device)
        torch.autograd.Variable._execution_engine.queue_callback(current)
    here = (g.device, _raw(g.device))
    last = current.writers.get(id(p), here)
    current.writers[id(p)] = here
    if last != here:
        torch.cuda.current_stream(g.device).wait_stream(_stream(*last))
    if current.left:
        _wait_for(current.left)
    if inner:
        current.inner.add(id(p))
    elif ready is not None:
        hooks = p._post_accumulate_grad_hooks
        if hooks is None or _accumulated not in hooks.values():
            p.register_post_accumulate_grad_hook(_accumulated)
    return True, g


def written(p) -> None:
    """After a write into ``p``'s flat gradient outside of any backward pass."""
    if _task() < 0:
        _native.grad_ready(p)


def refuse_twice(what: str) -> None:
    """Raised by a backward that runs with gradients recorded, which is what
    ``create_graph=True`` does: the kernels' gradients are not differentiable
    themselves and would count as constants."""
    raise RuntimeError(f"{what}: the gradient is not differentiable (create_graph=True)")
