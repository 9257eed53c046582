"""Layer normalisation over the last dimension (``csrc/kernels/layer_norm.hip``).

``layer_norm(x, weight, bias, eps)`` = ``(x - mean) / sqrt(var + eps) * weight +
bias`` with the (biased) statistics of each row in fp32, for fp32 / bf16 / fp16
inputs of any leading shape and row stride.  One launch forward; backward one
pass over the rows for ``dx`` and the column sums of ``dweight`` / ``dbias``
plus one launch that joins the sums in a fixed order (no atomics: results are
bit-reproducible).  Weight and bias gradients accumulate straight into the flat
fp32 gradient buffer when the parameter has one
(:func:`~zookeeper_amd.ops._native.direct_grad`).

``eps`` defaults to Keras' 1e-3, as in :class:`~zookeeper_amd.nn.BatchNorm`.
"""

from __future__ import annotations

import functools
from typing import Optional

import torch

from zookeeper_amd.ops._native import lib
from zookeeper_amd.ops._rows import (DTYPE_CODES, as_fp32, call, check_param, flat_grad, guard,
                                     in_backward, ptr, raw_stream, refuse_twice, rows_of, tracked,
                                     use_kernels, written)


@functools.lru_cache(maxsize=256)
def _ws_bytes(rows: int, cols: int) -> int:
    return lib().zk_layer_norm_bwd_ws_bytes(rows, cols)


def _forward(x, weight, bias, eps: float, stats: bool):
    """``y`` and the rows' mean and rstd ([2, rows] fp32, or None)."""
    x2, rows, stride = rows_of(x)
    dev = x.device
    y = torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype,
                                                                  device=dev)
    st = mean = rstd = None
    if stats:
        st = torch.empty((2, rows), dtype=torch.float32, device=dev)
        mean = st.data_ptr()
        rstd = mean + 4 * rows
    w, b = as_fp32(weight), as_fp32(bias)
    with guard(x):
        call(lib().zk_layer_norm_fwd, "zk_layer_norm_fwd", x2.data_ptr(), ptr(w), ptr(b),
             y.data_ptr(), mean, rstd, rows, int(x.shape[-1]), stride, eps, DTYPE_CODES[x.dtype],
             raw_stream(dev.index))
    return y, st


class _LayerNormFn(torch.autograd.Function):
    # Small rows wait for this host code and not for the kernels (a backward
    # runs on a cold thread): as few calls as possible.  The row stride is taken
    # anew: hooks on saved tensors may give ``x`` back in another layout.
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = _forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight)
        # the parameters themselves: the flat gradient buffer hangs on them
        ctx.rest = (stats, weight, bias, in_backward())
        return y

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():
            refuse_twice("layer_norm")
        x, weight = ctx.saved_tensors
        stats, wp, bp, inner = ctx.rest
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dev, cols = x.device, x.shape[-1]
        x2, rows, stride = rows_of(x)
        dx = ws = dw = db = dw_direct = db_direct = None
        add = ws_bytes = 0
        if dy.is_contiguous():
            dy2, dys = dy, cols
            if need_x:
                dx = torch.empty_like(dy)
        else:
            dy2, _, dys = rows_of(dy)
            if need_x:
                dx = torch.empty(x.shape, dtype=x.dtype, device=dev)
        L = lib()
        if need_w:
            need_w, dw_direct = flat_grad(ctx, wp, inner)
        if need_b:
            need_b, db_direct = flat_grad(ctx, bp, inner)
        if bp is wp:  # one buffer: two blocks would add to the same elements
            db_direct = None
        if need_w or need_b:
            new = torch.empty if rows else torch.zeros
            dw, db = dw_direct, db_direct
            if dw is not None:
                add = 1
            elif need_w:
                dw = new(cols, dtype=torch.float32, device=dev)
            if db is not None:
                add += 2
            elif need_b:
                db = new(cols, dtype=torch.float32, device=dev)
            ws_bytes = _ws_bytes(rows, cols)
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        if rows:
            mean = stats.data_ptr()
            w = as_fp32(weight)
            with guard(x):
                call(L.zk_layer_norm_bwd, "zk_layer_norm_bwd", dy2.data_ptr(), x2.data_ptr(),
                     ptr(w), mean, mean + 4 * rows, ptr(dx), ptr(dw), ptr(db), ptr(ws), ws_bytes,
                     rows, cols, stride, dys, DTYPE_CODES[x.dtype], add, raw_stream(dev.index))
        if dw_direct is not None:
            if bp is wp:
                dw_direct += db
                db = None
            written(wp)
            dw = None
        elif dw is not None and wp.dtype != torch.float32:
            dw = dw.to(wp.dtype)
        if db_direct is not None:
            written(bp)
            db = None
        elif db is not None and bp.dtype != torch.float32:
            db = db.to(bp.dtype)
        return dx, dw, db, None


def _plain(x, weight, bias, eps):
    """The same arithmetic in torch operations (host tensors), differentiable."""
    v = x if x.dtype == torch.float64 else x.float()
    c = v - v.mean(-1, keepdim=True)
    y = c * torch.rsqrt(c.square().mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.to(v.dtype)
    if bias is not None:
        y = y + bias.to(v.dtype)
    return y.to(x.dtype)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, eps: float = 1e-3) -> torch.Tensor:
    """Normalise the last dimension of ``x``; see the module docstring.

    ``weight`` / ``bias``: shape ``[x.shape[-1]]``, either may be None.  The
    result is contiguous and has ``x``'s type.  Raises ValueError for a 0-dim
    input, an empty last dimension, a negative ``eps``, types the kernels do not
    take and parameters of another shape or device."""
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"layer_norm: needs a non-empty last dimension, got {tuple(x.shape)}")
    if not eps >= 0.0:
        raise ValueError(f"layer_norm: eps must be >= 0, got {eps}")
    if weight is not None:
        check_param(weight, x.shape[-1], x, "layer_norm weight")
    if bias is not None:
        check_param(bias, x.shape[-1], x, "layer_norm bias")
    if not use_kernels(x, "layer_norm"):
        return _plain(x, weight, bias, eps)
    if x.shape[-1] >= 1 << 31 or x.numel() // x.shape[-1] >= 1 << 31:
        raise ValueError(f"layer_norm: at most 2^31 - 1 rows and columns, got {tuple(x.shape)}")
    if tracked() or torch.is_grad_enabled() and (
            x.requires_grad or (weight is not None and weight.requires_grad)
            or (bias is not None and bias.requires_grad)):
        return _LayerNormFn.apply(x, weight, bias, eps)
    return _forward(x, weight, bias, eps, False)[0]
