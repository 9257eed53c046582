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

from typing import Optional

import torch

from zookeeper_amd.ops._native import check, direct_grad, grad_ready, lib, stream_ptr
from zookeeper_amd.ops._rows import (DTYPE_CODES, as_fp32, check_param, guard, once_only, ptr,
                                     rows_of, use_kernels)


def _forward(x, weight, bias, eps: float, stats: bool):
    x2, rows, stride = rows_of(x)
    cols = x.shape[-1]
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    # [2, rows]: mean, rstd
    st = torch.empty((2, rows), dtype=torch.float32, device=x.device) if stats else None
    mean = st.data_ptr() if stats else None
    rstd = mean + 4 * rows if stats else None
    with guard(x):
        check(lib().zk_layer_norm_fwd(x2.data_ptr(), ptr(as_fp32(weight)), ptr(as_fp32(bias)),
                                      y.data_ptr(), mean, rstd, rows, cols, stride,
                                      eps, DTYPE_CODES[x.dtype], stream_ptr(x.device)),
              "zk_layer_norm_fwd")
    return y, st


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = _forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, stats)
        # the parameters themselves: the flat gradient buffer hangs on them
        ctx.weight_param, ctx.bias_param = weight, bias
        return y

    @staticmethod
    def backward(ctx, dy):
        once_only("layer_norm")
        x, weight, stats = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        wp, bp = ctx.weight_param, ctx.bias_param
        dev, cols = x.device, x.shape[-1]
        dw_direct = direct_grad(wp) if need_w else None
        db_direct = direct_grad(bp) if need_b else None
        x2, rows, xs = rows_of(x)
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_x else None
        if rows == 0:
            dw = torch.zeros_like(wp) if need_w and dw_direct is None else None
            db = torch.zeros_like(bp) if need_b and db_direct is None else None
        else:
            dy2, _, dys = rows_of(dy)
            dw, db = dw_direct, db_direct
            if need_w and dw is None:
                dw = torch.empty(cols, dtype=torch.float32, device=dev)
            if need_b and db is None:
                db = torch.empty(cols, dtype=torch.float32, device=dev)
            ws, ws_bytes = None, 0
            if need_w or need_b:
                ws_bytes = lib().zk_layer_norm_bwd_ws_bytes(rows, cols)
                ws = torch.empty(ws_bytes // 4, dtype=torch.float32, device=dev)
            add = (1 if dw_direct is not None else 0) | (2 if db_direct is not None else 0)
            with guard(x):
                check(lib().zk_layer_norm_bwd(dy2.data_ptr(), x2.data_ptr(), ptr(as_fp32(weight)),
                                              stats.data_ptr(), stats.data_ptr() + 4 * rows,
                                              ptr(dx), ptr(dw),
                                              ptr(db), ptr(ws), ws_bytes, rows, cols, xs, dys,
                                              DTYPE_CODES[x.dtype], add, stream_ptr(dev)),
                      "zk_layer_norm_bwd")
        if dw_direct is not None:
            grad_ready(wp)
            dw = None
        elif dw is not None and dw.dtype != wp.dtype:
            dw = dw.to(wp.dtype)
        if db_direct is not None:
            grad_ready(bp)
            db = None
        elif db is not None and db.dtype != bp.dtype:
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
    if torch.is_grad_enabled() and (x.requires_grad
                                    or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _LayerNormFn.apply(x, weight, bias, eps)
    return _forward(x, weight, bias, eps, False)[0]
