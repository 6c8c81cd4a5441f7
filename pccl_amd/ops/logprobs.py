"""Log probabilities of given tokens, with the row's entropy and its top alternatives, differentiable.

The loss of a language model (``-logprob.mean()``), its evaluation and the scoring of sampled tokens in one pass over
the logits in their own type: no fp32 copy, no log-softmax tensor. GPU tensors run the HIP kernels
(csrc/hip/hip_logprob.hip) on the current stream without synchronising; CPU tensors run plain torch operations.
"""
from __future__ import annotations

from operator import index
from typing import NamedTuple, Optional

import torch

from .._native import C
from ._launch import on_device, refuse_tangents, require_hip, stream_of
from .kernels import WIRE_DTYPE, _check

MAX_TOP_LOGPROBS = 64


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor                 # fp32, logits.shape[:-1]; 0 where the target is ignore_index
    entropy: torch.Tensor                 # fp32, logits.shape[:-1]
    top_logprob: Optional[torch.Tensor]   # fp32, logits.shape[:-1] + (top_k,), falling; None for top_k = 0
    top_index: Optional[torch.Tensor]     # int64, the alternatives' tokens


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _rows(logits: torch.Tensor, targets: torch.Tensor):
    """[rows, vocab] with the vocabulary contiguous and the targets in one run: views where the strides allow it, else
    copies. (Tensors that are so already are not touched: the backward pass runs this on the autograd thread, where
    every call into torch costs several microseconds.)"""
    x = logits if logits.dim() == 2 else logits.reshape(-1, logits.shape[-1])
    if x.stride(1) != 1 and x.shape[1] != 1:
        x = x.contiguous()
    t = targets if targets.dim() == 1 else targets.reshape(-1)
    return x, t if t.is_contiguous() else t.contiguous()


def _host_forward(x: torch.Tensor, targets: torch.Tensor, top_k: int, ignore_index: int):
    xf = x.float()
    m = xf.masked_fill(xf.isnan(), -torch.inf).amax(dim=1)
    mu = torch.where(m == -torch.inf, 0.0, m)
    d = xf - mu[:, None]
    e = d.exp()
    s = e.sum(dim=1)
    empty = (m == -torch.inf) & (s == 0)
    log_s = torch.where(empty, 0.0, s.log())
    entropy = torch.where(empty, 0.0, log_s - (e * d.clamp(min=-200.0)).sum(dim=1) / s)
    stats = torch.stack([m, log_s, entropy], dim=1)
    logp = torch.where(empty[:, None], -torch.inf, (xf - m[:, None]) - log_s[:, None])
    known = (targets >= 0) & (targets < x.shape[1])
    lp = logp.gather(1, torch.where(known, targets, 0)[:, None])[:, 0]
    logprob = torch.where(targets == ignore_index, 0.0, torch.where(known, lp, torch.nan))
    top_lp = top_ix = None
    if top_k:
        order = xf.masked_fill(xf.isnan(), -torch.inf)
        top_ix = order.sort(dim=1, descending=True, stable=True).indices[:, :top_k].contiguous()
        top_lp = logp.gather(1, top_ix)
    return logprob, entropy, stats, top_lp, top_ix


def _host_backward(x, targets, ignore_index, stats, top_ix, g_lp, g_h, g_top):
    m, log_s, entropy = stats.split(1, dim=1)
    empty = (m == -torch.inf) & (log_s == 0)
    logp = (x.float() - m) - log_s
    zero = torch.zeros_like(entropy[:, 0])
    used = targets != ignore_index
    known = (targets >= 0) & (targets < x.shape[1])
    gs = zero if g_lp is None else torch.where(used, torch.where(known, g_lp, torch.nan), 0.0)
    at_target = zero if g_lp is None else torch.where(used & known, g_lp, 0.0)
    if g_top is not None:
        gs = gs + g_top.sum(dim=1)
    term = gs[:, None]
    if g_h is not None:
        term = term + g_h[:, None] * (logp.clamp(min=-200.0) + entropy)
    d = -logp.exp() * term
    d.scatter_add_(1, torch.where(known, targets, 0)[:, None], at_target[:, None])
    if g_top is not None:
        d.scatter_add_(1, top_ix, g_top)
    return torch.where(empty, 0.0, d).to(x.dtype)


def _device_forward(x: torch.Tensor, targets: torch.Tensor, top_k: int, ignore_index: int):
    n, v = x.shape
    device = x.device
    logprob = torch.empty(n, dtype=torch.float32, device=device)
    entropy = torch.empty(n, dtype=torch.float32, device=device)
    stats = torch.empty((n, 3), dtype=torch.float32, device=device)
    top_lp = top_ix = None
    if top_k:
        top_lp = torch.empty((n, top_k), dtype=torch.float32, device=device)
        top_ix = torch.empty((n, top_k), dtype=torch.int64, device=device)
    _check(C.pcclxTokenLogprobs(x.data_ptr(), x.stride(0), n, v, WIRE_DTYPE[x.dtype], targets.data_ptr(),
                                ignore_index, top_k, logprob.data_ptr(), entropy.data_ptr(), stats.data_ptr(),
                                _ptr(top_lp), _ptr(top_ix), stream_of(device)), "token_logprobs")
    return logprob, entropy, stats, top_lp, top_ix


def _device_backward(x, targets, ignore_index, stats, top_ix, g_lp, g_h, g_top):
    n, v = x.shape
    d = x.new_empty((n, v))
    if g_lp is not None and not g_lp.is_contiguous():
        g_lp = g_lp.contiguous()
    if g_h is not None and not g_h.is_contiguous():
        g_h = g_h.contiguous()
    if g_top is not None and not g_top.is_contiguous():
        g_top = g_top.contiguous()
    _check(C.pcclxTokenLogprobsGrad(x.data_ptr(), x.stride(0), n, v, WIRE_DTYPE[x.dtype], targets.data_ptr(),
                                    ignore_index, 0 if top_ix is None else top_ix.shape[-1], stats.data_ptr(),
                                    _ptr(top_ix), _ptr(g_lp), _ptr(g_h), _ptr(g_top), d.data_ptr(),
                                    stream_of(x.device)), "token_logprobs_grad")
    return d


def _forward(logits: torch.Tensor, targets: torch.Tensor, top_k: int, ignore_index: int):
    shape = targets.shape
    x, t = _rows(logits, targets)
    if x.is_cuda:
        with on_device(x.device):
            logprob, entropy, stats, top_lp, top_ix = _device_forward(x, t, top_k, ignore_index)
    else:
        logprob, entropy, stats, top_lp, top_ix = _host_forward(x, t, top_k, ignore_index)
    if len(shape) != 1:
        logprob, entropy = logprob.view(shape), entropy.view(shape)
        if top_k:
            top_lp, top_ix = top_lp.view(shape + (top_k,)), top_ix.view(shape + (top_k,))
    return logprob, entropy, stats, top_lp, top_ix


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top_k, ignore_index):
        logprob, entropy, ctx.stats, top_lp, top_ix = _forward(logits, targets, top_k, ignore_index)
        if top_k:
            ctx.mark_non_differentiable(top_ix)
        ctx.ignore_index = ignore_index
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, targets, top_ix)
        return logprob, entropy, top_lp, top_ix

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_lp, g_h, g_top, _):
        logits, targets, top_ix = ctx.saved_tensors
        if g_lp is None and g_h is None and g_top is None:
            return None, None, None, None
        x, t = _rows(logits, targets)
        if logits.dim() != 2:
            g_lp, g_h = (None if g is None else g.reshape(-1) for g in (g_lp, g_h))
            top_ix, g_top = (None if v is None else v.reshape(-1, v.shape[-1]) for v in (top_ix, g_top))
        if x.is_cuda:
            with on_device(x.device):
                d = _device_backward(x, t, ctx.ignore_index, ctx.stats, top_ix, g_lp, g_h, g_top)
        else:
            d = _host_backward(x, t, ctx.ignore_index, ctx.stats, top_ix, g_lp, g_h, g_top)
        return d if logits.dim() == 2 else d.view(logits.shape), None, None, None


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, *, top_k: int = 0,
                   ignore_index: int = -100) -> TokenLogprobs:
    """Log probability of ``targets`` under ``softmax(logits)``, the entropy of that distribution, and its ``top_k``
    most likely tokens.

    ``logits``: fp32 / bf16 / fp16, any leading shape and strides (the vocabulary should be contiguous: other layouts
    are copied). ``targets``: int64, ``logits.shape[:-1]``, on the same device. Results are fp32, sums in fp32; equal
    calls give equal bits. ``top_k`` at most 64; equal logits rank by the lower index, NaN with ``-inf``.

    * targets equal to ``ignore_index`` have log probability 0 and no gradient through it;
    * a target outside the vocabulary has log probability NaN, and NaN gradients (checking it would wait for the GPU);
    * ``-inf`` logits are masked tokens: probability 0, no share in the entropy, gradient 0; only a masked
      target or alternative, of log probability ``-inf``, gets its upstream gradient (times 1 - p = 1);
    * a row whose every logit is ``-inf`` has entropy 0, log probabilities ``-inf`` and gradient 0;
    * a row with a NaN or ``+inf`` has NaN results and gradients.

    ``logprob``, ``entropy`` and ``top_logprob`` are differentiable with respect to ``logits``, once and in backward
    mode (logits on a GPU with a forward-mode tangent are refused). The call and its backward only queue kernels, so both
    may be captured into a graph. (Before a backward pass is captured, drop the results of eager calls on the same
    leaves: torch ends the process when their graph is still alive.)
    """
    top_k, ignore_index = index(top_k), index(ignore_index)
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"token_logprobs: logits need a vocabulary dimension, got shape {tuple(logits.shape)}")
    if logits.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError(f"token_logprobs: logits must be fp32/bf16/fp16, got {logits.dtype}")
    if targets.dtype != torch.int64:
        raise TypeError(f"token_logprobs: targets must be int64, got {targets.dtype}")
    if targets.shape != logits.shape[:-1]:
        raise ValueError(f"token_logprobs: targets of shape {tuple(targets.shape)} do not match logits of shape "
                         f"{tuple(logits.shape)}")
    if targets.device != logits.device:
        raise ValueError(f"token_logprobs: targets on {targets.device}, logits on {logits.device}")
    if not 0 <= top_k <= min(MAX_TOP_LOGPROBS, logits.shape[-1]):
        raise ValueError(f"token_logprobs: top_k {top_k} is not in 0..{min(MAX_TOP_LOGPROBS, logits.shape[-1])}")
    if not -1 << 63 <= ignore_index < 1 << 63:  # the kernels would take it modulo 2^64
        raise ValueError(f"token_logprobs: ignore_index {ignore_index} is no int64")
    if targets.numel() >= 1 << 31 or logits.shape[-1] >= 1 << 31:
        raise ValueError("token_logprobs: at most 2^31 - 1 rows and tokens of vocabulary")
    if logits.device.type == "cuda":
        require_hip()
        refuse_tangents("token_logprobs", logits)
    elif logits.device.type != "cpu":
        raise ValueError(f"token_logprobs: no kernel for device {logits.device}")
    if logits.requires_grad and torch.is_grad_enabled():
        return TokenLogprobs(*_TokenLogprobs.apply(logits, targets, top_k, ignore_index))
    logprob, entropy, _, top_lp, top_ix = _forward(logits, targets, top_k, ignore_index)
    return TokenLogprobs(logprob, entropy, top_lp, top_ix)
