"""Log probabilities of given tokens (classes), the entropy of each row and its
most likely alternatives (``csrc/kernels/logprobs.hip``).

``token_logprobs(logits, tokens, top=k)`` takes rows of fp32 / bf16 / fp16 logits
``[..., V]`` (any row stride) and returns fp32 values of shape ``[...]``: the log
probability of each given token, the entropy of the row's distribution in nats,
and with ``top > 0`` the log probabilities and places of the ``top`` greatest
logits, greatest first, the lower place first among equals.

Log probability and entropy are differentiable in the logits (policy losses,
distillation, entropy bonuses); one pass over the logits forward, one backward.
The alternatives are for reporting and carry no gradient.

* A token equal to ``ignore_index`` (inside ``[0, V)`` or not) gives log
  probability 0 without gradient; the row's entropy is not affected.
* Masked logits are ``-inf``: probability 0, no share in the entropy.  A row of
  nothing but ``-inf`` has log probability ``-inf``, entropy 0, gradient 0.
* Any other token outside ``[0, V)`` gives a log probability of NaN, whose gradient
  makes the row's NaN; the entropy and its gradient do not depend on the token.
* A row with a NaN or ``+inf`` gives NaN for both and a NaN gradient row (a NaN ranks
  above all numbers among the alternatives).
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from zookeeper_amd.ops._native import lib
from zookeeper_amd.ops._rows import (DTYPE_CODES, call, guard, ptr, raw_stream, refuse_twice,
                                     rows_of, tracked, use_kernels)

MAX_TOP = 64


class TokenLogProbs(NamedTuple):
    logp: torch.Tensor
    entropy: torch.Tensor
    top_logp: Optional[torch.Tensor] = None
    top_ids: Optional[torch.Tensor] = None


def _forward(logits, tokens, top: int, ignore: int, keep: bool):
    dev, lead, V = logits.device, logits.shape[:-1], int(logits.shape[-1])
    x, rows, stride = rows_of(logits)
    L = lib()
    f32 = torch.float32
    logp = torch.empty(lead, dtype=f32, device=dev)
    entropy = torch.empty(lead, dtype=f32, device=dev)
    stats = torch.empty((rows, 3), dtype=f32, device=dev) if keep else None
    top_logp = top_ids = ws = None
    if top:
        top_logp = torch.empty((*lead, top), dtype=f32, device=dev)
        top_ids = torch.empty((*lead, top), dtype=torch.int64, device=dev)
    ws_bytes = L.zk_token_logprobs_ws_bytes(rows, V, top)
    if ws_bytes:
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    with guard(logits):
        call(L.zk_token_logprobs_fwd, "zk_token_logprobs_fwd", x.data_ptr(), tokens.data_ptr(),
             logp.data_ptr(), entropy.data_ptr(), ptr(stats), ptr(top_logp), ptr(top_ids),
             ptr(ws), ws_bytes, rows, V, stride, top, ignore, DTYPE_CODES[logits.dtype],
             raw_stream(dev.index))
    return logp, entropy, top_logp, top_ids, stats


class _TokenLogProbsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top, ignore):
        logp, entropy, top_logp, top_ids, stats = _forward(logits, tokens, top, ignore, True)
        ctx.save_for_backward(logits, tokens)
        ctx.rest = (stats, ignore)
        ctx.set_materialize_grads(False)
        if top:
            ctx.mark_non_differentiable(top_logp, top_ids)
            return logp, entropy, top_logp, top_ids
        return logp, entropy

    @staticmethod
    def backward(ctx, g_logp, g_entropy, *_):
        if torch.is_grad_enabled():
            refuse_twice("token_logprobs")
        if g_logp is None and g_entropy is None:
            return None, None, None, None
        logits, tokens = ctx.saved_tensors
        stats, ignore = ctx.rest
        # anew: hooks on saved tensors may change the layout
        x, rows, stride = rows_of(logits)
        tokens = tokens.contiguous()
        if logits.is_contiguous():
            dx = torch.empty_like(logits)
        else:
            dx = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        if g_logp is not None and not g_logp.is_contiguous():
            g_logp = g_logp.contiguous()
        if g_entropy is not None and not g_entropy.is_contiguous():
            g_entropy = g_entropy.contiguous()
        with guard(logits):
            call(lib().zk_token_logprobs_bwd, "zk_token_logprobs_bwd", x.data_ptr(),
                 tokens.data_ptr(), stats.data_ptr(), ptr(g_logp), ptr(g_entropy), dx.data_ptr(),
                 rows, logits.shape[-1], stride, ignore, DTYPE_CODES[logits.dtype],
                 raw_stream(logits.device.index))
        return dx, None, None, None


def _plain(logits, tokens, top, ignore):
    """The same in torch operations (host tensors), differentiable."""
    x = logits if logits.dtype == torch.float64 else logits.float()
    V = x.shape[-1]
    gone = torch.isneginf(x).all(-1, keepdim=True)
    lp = torch.log_softmax(torch.where(gone, torch.zeros_like(x), x), -1)
    p = lp.exp()
    masked = p == 0  # 0 ln 0 = 0
    entropy = -(p * torch.where(masked, torch.zeros_like(lp), lp)).sum(-1)
    entropy = torch.where(gone[..., 0], torch.zeros_like(entropy), entropy)
    lp = torch.where(gone, torch.full_like(lp, float("-inf")), lp)
    logp = lp.gather(-1, tokens.clamp(0, V - 1).unsqueeze(-1))[..., 0]
    # a token out of range: NaN with a NaN gradient; an ignored one: 0 without
    bad = ((tokens < 0) | (tokens >= V)) & (tokens != ignore)
    logp = logp * torch.where(bad, float("nan"), 1.0).to(lp.dtype)
    logp = torch.where(tokens == ignore, torch.zeros_like(logp), logp)
    if not top:
        return TokenLogProbs(logp, entropy)
    ids = x.detach().sort(stable=True, dim=-1, descending=True).indices[..., :top]
    return TokenLogProbs(logp, entropy, lp.detach().gather(-1, ids), ids)


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0,
                   ignore_index: int = -100) -> TokenLogProbs:
    """Log probabilities, entropies and alternatives; see the module docstring.

    ``tokens``: whole numbers of ``logits``' leading shape on its device; ``0 <=
    top <= min(V, 64)``.  Raises ValueError otherwise, for an empty last
    dimension and for types the kernels do not take."""
    if logits.dim() == 0 or logits.shape[-1] == 0:
        raise ValueError(f"token_logprobs: needs a non-empty last dimension, "
                         f"got {tuple(logits.shape)}")
    if tokens.shape != logits.shape[:-1]:
        raise ValueError(f"token_logprobs: tokens of shape {tuple(logits.shape[:-1])} expected, "
                         f"got {tuple(tokens.shape)}")
    if tokens.dtype != torch.int64:
        if tokens.dtype not in (torch.int32, torch.int16, torch.uint8, torch.int8):
            raise ValueError(f"token_logprobs: tokens must be whole numbers, got {tokens.dtype}")
        tokens = tokens.to(torch.int64)
    if tokens.device != logits.device:
        raise ValueError(f"token_logprobs: tokens on {tokens.device}, logits on {logits.device}")
    top = int(top)
    if not 0 <= top <= min(MAX_TOP, logits.shape[-1]):
        raise ValueError(f"token_logprobs: top must be in [0, {min(MAX_TOP, logits.shape[-1])}], "
                         f"got {top}")
    if not -2 ** 63 <= ignore_index < 2 ** 63:
        raise ValueError(f"token_logprobs: ignore_index {ignore_index} is no 64-bit number")
    if not use_kernels(logits, "token_logprobs"):
        return _plain(logits, tokens, top, ignore_index)
    if logits.shape[-1] >= 0x7FFF0000:
        raise ValueError(f"token_logprobs: rows of {logits.shape[-1]} elements are too long")
    tokens = tokens.contiguous()
    if tracked() or logits.requires_grad and torch.is_grad_enabled():
        return TokenLogProbs(*_TokenLogProbsFn.apply(logits, tokens, top, ignore_index))
    return TokenLogProbs(*_forward(logits, tokens, top, ignore_index, False)[:4])
