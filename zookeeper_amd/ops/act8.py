"""Activations kept in 8 bits for the backward pass (``csrc/kernels/act8.hip``).

What a layer saves for its backward pass is most of a training step's memory;
here it is one signed byte per value and one scale byte per 32 instead of 2 or 4
bytes per value.

* :func:`pack8` / :func:`unpack8` -- the form itself (:class:`Packed8`): blocks
  of 32 values along the last dimension share a power-of-two step, every value
  is within half a step of what it stands for, and half a step is at most 1 /
  127.5 of the block's largest value (or 2^-127).  A block with an infinity or a NaN stands for
  NaN.
* :func:`gelu8` -- GELU (the exact form ``x * Phi(x)``) that keeps its input in 8
  bits; the same pass over ``x`` writes the output and the kept form.
* :func:`dense8` -- a dense layer that keeps its input in 8 bits; its weight
  gradient ``dy^T x8`` and bias gradient come from :func:`dense8_grads`, a matrix
  product that decodes the kept input on its way to the matrix units.

Forward results are exact (they use the unrounded input); gradients are those
of the kept input.  ``dense8`` computes ``y`` and ``dx`` with the library's
matrix products, like the framework's other dense layers.  Host tensors run the
same definitions in PyTorch.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
import torch.nn.functional as F

from zookeeper_amd.ops._native import lib
from zookeeper_amd.ops._rows import (DTYPE_CODES, call, flat_grad, guard, in_backward, ptr,
                                     raw_stream, refuse_tracing, refuse_twice, rows_of, tracked,
                                     use_kernels, written)

BLOCK = 32


class Packed8:
    """The 8-bit form of a tensor: ``codes`` int8 of its shape, ``scales`` uint8
    with a last dimension of ``ceil(n / 32)``; a value is ``code * 2^(scale -
    133)``, scale 255 stands for NaN.  ``dtype``: the packed tensor's type."""

    __slots__ = ("codes", "scales", "dtype")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype):
        want = (*codes.shape[:-1], -(-codes.shape[-1] // BLOCK)) if codes.dim() else None
        if (codes.dtype != torch.int8 or scales.dtype != torch.uint8 or want is None
                or tuple(scales.shape) != want or codes.device != scales.device
                or not codes.is_contiguous() or not scales.is_contiguous()
                or not dtype.is_floating_point):
            raise ValueError(
                "Packed8: expected contiguous int8 codes [..., n] and uint8 scales "
                f"[..., ceil(n / {BLOCK})] on one device, got {codes.dtype} {tuple(codes.shape)} "
                f"and {scales.dtype} {tuple(scales.shape)}")
        self.codes, self.scales, self.dtype = codes, scales, dtype

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def __repr__(self) -> str:
        return f"Packed8(shape={tuple(self.shape)}, dtype={self.dtype}, device={self.device})"


def _check_input(x: torch.Tensor, what: str) -> None:
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"{what}: needs a non-empty last dimension, got {tuple(x.shape)}")


def _empty_form(x):
    codes = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scales = torch.empty((*x.shape[:-1], -(-int(x.shape[-1]) // BLOCK)), dtype=torch.uint8,
                         device=x.device)
    return codes, scales


# --- the definitions in PyTorch (host tensors) --------------------------------

def _steps(scales):
    """2^(scale - 133) of each block, fp32 (subnormal under 7); NaN for 255."""
    s = scales.to(torch.int32)
    low = torch.ones_like(s) << (s.clamp_max(6) + 16)
    step = torch.where(s < 7, low, (s - 6) << 23).view(torch.float32)
    return torch.where(s == 255, torch.full_like(step, float("nan")), step)


def _pack_plain(x):
    n = x.shape[-1]
    v = F.pad(x.detach().float(), (0, -n % BLOCK)).unflatten(-1, (-1, BLOCK))
    top = v.abs().amax(-1)  # NaN if the block holds one
    fine = torch.isfinite(top)
    top = torch.where(fine, top, torch.ones_like(top))
    e = (top.contiguous().view(torch.int32) >> 23).clamp_min(7)
    inv = ((260 - e) << 23).view(torch.float32)
    e = e + (((top * inv).round() >= 128) & (e < 254)).to(torch.int32)
    inv = ((260 - e) << 23).view(torch.float32)
    codes = (v * inv.unsqueeze(-1)).round().clamp(-127, 127)
    codes = torch.where(fine.unsqueeze(-1), codes, torch.zeros_like(codes))
    e = torch.where(fine, e, torch.full_like(e, 255))
    return (codes.to(torch.int8).flatten(-2)[..., :n].contiguous(), e.to(torch.uint8).contiguous())


def _unpack_plain(codes, scales, dtype):
    n = codes.shape[-1]
    step = _steps(scales).repeat_interleave(BLOCK, -1)[..., :n]
    return (codes.float() * step).to(dtype)


def _gelu_slope(k):
    return (0.5 * torch.erfc(k * -math.sqrt(0.5))
            + k * torch.exp(-0.5 * k * k) * (1 / math.sqrt(2 * math.pi)))


# --- pack / unpack --------------------------------------------------------------

def _pack(x):
    codes, scales = _empty_form(x)
    x2, rows, stride = rows_of(x)
    with guard(x):
        call(lib().zk_pack8, "zk_pack8", x2.data_ptr(), codes.data_ptr(), scales.data_ptr(), rows,
             int(x.shape[-1]), stride, DTYPE_CODES[x.dtype], raw_stream(x.device.index))
    return codes, scales


def pack8(x: torch.Tensor) -> Packed8:
    """The 8-bit form of ``x`` (fp32, bf16 or fp16 on the GPU; any leading shape
    and row stride).  Not differentiable: the form is what a backward keeps."""
    _check_input(x, "pack8")
    if not use_kernels(x, "pack8"):
        return Packed8(*_pack_plain(x), x.dtype)
    refuse_tracing("pack8")
    return Packed8(*_pack(x), x.dtype)


def unpack8(kept: Packed8, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The values that ``kept`` stands for, in ``dtype`` (default: the packed
    tensor's type).  Exact in bf16 and fp32."""
    dtype = kept.dtype if dtype is None else dtype
    out = torch.empty(kept.shape, dtype=dtype, device=kept.device)
    if not use_kernels(out, "unpack8"):
        return _unpack_plain(kept.codes, kept.scales, dtype)
    refuse_tracing("unpack8")
    if out.numel() == 0:
        return out
    n = kept.shape[-1]
    with guard(out):
        call(lib().zk_unpack8, "zk_unpack8", kept.codes.data_ptr(), kept.scales.data_ptr(),
             out.data_ptr(), out.numel() // n, n, DTYPE_CODES[dtype],
             raw_stream(out.device.index))
    return out


# --- GELU -------------------------------------------------------------------------

def _gelu_forward(x, keep: bool):
    """``y`` and the kept input in one buffer: the codes, then the scales."""
    x2, rows, stride = rows_of(x)
    n = int(x.shape[-1])
    dev = x.device
    y = torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype,
                                                                  device=dev)
    kept = codes = scales = None
    if keep:
        kept = torch.empty(rows * (n + (n + BLOCK - 1) // BLOCK), dtype=torch.uint8, device=dev)
        codes = kept.data_ptr()
        scales = codes + rows * n
    with guard(x):
        call(lib().zk_gelu8_fwd, "zk_gelu8_fwd", x2.data_ptr(), y.data_ptr(), codes, scales, rows,
             n, stride, DTYPE_CODES[x.dtype], raw_stream(dev.index))
    return y, kept, rows


class _Gelu8Fn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        y, kept, ctx.rows = _gelu_forward(x, True)
        ctx.save_for_backward(kept)
        return y

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():
            refuse_twice("gelu8")
        kept = ctx.saved_tensors[0].contiguous()  # hooks may have changed the layout
        n, rows, dev = dy.shape[-1], ctx.rows, dy.device
        if dy.is_contiguous():
            dx, dy2, stride = torch.empty_like(dy), dy, n
        else:
            dx = torch.empty(dy.shape, dtype=dy.dtype, device=dev)
            dy2, _, stride = rows_of(dy)
        codes = kept.data_ptr()
        with guard(dy):
            call(lib().zk_gelu8_bwd, "zk_gelu8_bwd", dy2.data_ptr(), codes, codes + rows * n,
                 dx.data_ptr(), rows, n, stride, DTYPE_CODES[dy.dtype], raw_stream(dev.index))
        return dx


class _Gelu8HostFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        ctx.save_for_backward(*_pack_plain(x))
        return F.gelu(x)

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():
            refuse_twice("gelu8")
        k = _unpack_plain(*ctx.saved_tensors, torch.float32).to(
            torch.float64 if dy.dtype == torch.float64 else torch.float32)
        return (dy.to(k.dtype) * _gelu_slope(k)).to(dy.dtype)


def gelu8(x: torch.Tensor) -> torch.Tensor:
    """``x * Phi(x)``; the input is kept in 8 bits for the backward (nothing is
    kept when no gradient is wanted).  See the module docstring."""
    _check_input(x, "gelu8")
    native = use_kernels(x, "gelu8")
    if x.requires_grad and torch.is_grad_enabled():
        return _Gelu8Fn.apply(x) if native else _Gelu8HostFn.apply(x)
    if not native:
        return F.gelu(x)
    return _Gelu8Fn.apply(x) if tracked() else _gelu_forward(x, False)[0]


# --- dense ------------------------------------------------------------------------

def _dense_grads(dy, codes, scales, want_b: bool, dw=None, db=None, variant: int = -1):
    """fp32 ``dw`` [N, K] and ``db`` [N] of ``dy`` [..., N] and the kept input
    [..., K]; given ``dw`` / ``db`` buffers are added to.  ``variant`` picks a
    kernel (-1: by size)."""
    N, K = dy.shape[-1], codes.shape[-1]
    dev = dy.device
    dy2, rows, stride = rows_of(dy)
    if stride >= 1 << 24:  # the kernels' row offsets are 32-bit
        dy2, stride = dy2.contiguous(), N
    add = (1 if dw is not None else 0) | (2 if db is not None else 0)
    new = torch.zeros if rows == 0 else torch.empty
    if dw is None:
        dw = new((N, K), dtype=torch.float32, device=dev)
    if want_b and db is None:
        db = new((N,), dtype=torch.float32, device=dev)
    if rows == 0:
        return dw, db
    L = lib()
    dt = DTYPE_CODES[dy.dtype]
    ws_bytes = L.zk_dense8_wgrad_ws_bytes(rows, N, K, stride, dt, dy2.data_ptr() % 16 == 0,
                                          variant)
    if ws_bytes < 0:
        raise ValueError(f"dense8: sizes rows={rows}, outputs={N}, inputs={K} are not supported")
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    with guard(dy):
        call(L.zk_dense8_wgrad, "zk_dense8_wgrad", dy2.data_ptr(), codes.data_ptr(),
             scales.data_ptr(), dw.data_ptr(), ptr(db) if want_b else None, ws.data_ptr(),
             ws_bytes, rows, N, K, stride, dt, add, variant, raw_stream(dev.index))
    return dw, db


def dense8_grads(dy: torch.Tensor, kept: Packed8,
                 bias: bool = True) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``(dw, db)`` of a dense layer ``y = x w^T + b`` in fp32: ``dw`` [N, K] =
    ``dy^T x8`` and ``db`` [N] = the sum of ``dy`` over its rows (None without
    ``bias``), from the output gradient ``dy`` [..., N] (fp32, bf16 or fp16, any
    row stride) and the kept input [..., K].

    bf16 gradients take one matrix product, fp16 and fp32 gradients two and
    three (their exact bf16 terms); sums are fp32 in a fixed order.  Not
    differentiable."""
    _check_input(dy, "dense8_grads")
    if dy.shape[:-1] != kept.shape[:-1]:
        raise ValueError(f"dense8_grads: rows differ: dy {tuple(dy.shape)}, "
                         f"kept input {tuple(kept.shape)}")
    if dy.device != kept.device:
        raise ValueError(f"dense8_grads: dy on {dy.device}, the kept input on {kept.device}")
    dy = dy.detach()
    if use_kernels(dy, "dense8_grads"):
        refuse_tracing("dense8_grads")
        return _dense_grads(dy, kept.codes, kept.scales, bias)
    d = dy.reshape(-1, dy.shape[-1]).float()
    x = _unpack_plain(kept.codes, kept.scales, torch.float32).reshape(-1, kept.shape[-1])
    return d.t() @ x, d.sum(0) if bias else None


def _product(f, x, *operands):
    """``f(x, *operands)`` with the rows of ``x`` as one matrix.  torch makes a batched
    product of rows that do not merge, with a transposed view as its right operand, a
    form that has faulted in bfloat16."""
    if x.dim() <= 2:
        return f(x, *operands)
    return f(x.reshape(-1, x.shape[-1]), *operands).unflatten(0, x.shape[:-1])


def _linear(x, weight, bias):
    return _product(F.linear, x, weight.to(x.dtype), bias.to(x.dtype) if bias is not None else None)


class _Dense8Fn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        y = _linear(x, weight, bias)
        codes = scales = None
        if ctx.needs_input_grad[1]:
            codes, scales = _pack(x) if use_kernels(x, "dense8") else _pack_plain(x)
        ctx.save_for_backward(codes, scales, weight)
        ctx.weight_param, ctx.bias_param = weight, bias
        ctx.inner = in_backward()
        return y

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():
            refuse_twice("dense8")
        codes, scales, weight = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad
        wp, bp = ctx.weight_param, ctx.bias_param
        dx = _product(torch.matmul, dy, weight.to(dy.dtype)) if need_x else None
        dw = db = None
        native = use_kernels(dy, "dense8")
        dw_direct = db_direct = None
        if need_w and native:
            need_w, dw_direct = flat_grad(ctx, wp, ctx.inner)
        if need_b and native:
            need_b, db_direct = flat_grad(ctx, bp, ctx.inner)
        if need_w and native:  # contiguous: hooks may have changed the layout
            dw, db = _dense_grads(dy, codes.contiguous(), scales.contiguous(), need_b, dw_direct,
                                  db_direct)
        elif need_w:
            dw, db = dense8_grads(dy, Packed8(codes.contiguous(), scales.contiguous(), dy.dtype),
                                  need_b)
        elif need_b and native:  # a frozen weight with a trainable bias: of a column of zeros
            none = torch.zeros((dy.numel() // dy.shape[-1], 1), dtype=torch.int8, device=dy.device)
            _, db = _dense_grads(dy, none, none.view(torch.uint8), True, None, db_direct)
        elif need_b:
            db = dy.reshape(-1, dy.shape[-1]).float().sum(0)
        if dw_direct is not None:
            written(wp)
            dw = None
        elif dw is not None:
            dw = dw.to(wp.dtype)
        if db_direct is not None:
            written(bp)
            db = None
        elif db is not None:
            db = db.to(bp.dtype)
        return dx, dw, db


def dense8(x: torch.Tensor, weight: torch.Tensor,
           bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x weight^T + bias`` in ``x``'s type, its input kept in 8 bits for the
    weight gradient; see the module docstring.  ``weight`` [N, K], ``bias`` [N]
    of any floating type (their gradients have it; flat fp32 gradient buffers
    are accumulated into directly)."""
    _check_input(x, "dense8")
    if weight.dim() != 2 or weight.shape[1] != x.shape[-1] or weight.shape[0] == 0:
        raise ValueError(f"dense8: weight of shape (outputs, {x.shape[-1]}) expected, "
                         f"got {tuple(weight.shape)}")
    if bias is not None and tuple(bias.shape) != (weight.shape[0],):
        raise ValueError(f"dense8: bias of shape ({weight.shape[0]},) expected, "
                         f"got {tuple(bias.shape)}")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None and (p.device != x.device or not p.is_floating_point()):
            raise ValueError(f"dense8: {name} must be a floating-point tensor on {x.device}, "
                             f"got {p.dtype} on {p.device}")
    use_kernels(x, "dense8")
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad
                                    or (bias is not None and bias.requires_grad)):
        return _Dense8Fn.apply(x, weight, bias)
    return _linear(x, weight, bias)
