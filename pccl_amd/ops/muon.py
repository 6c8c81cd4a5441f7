"""Newton-Schulz orthogonalisation, and the Muon optimiser step built on it.

Muon replaces the momentum update U of a weight matrix by its orthogonal factor, approximated by a few steps of
``X <- a X + (b A + c A A) X`` with ``A = X X^T`` from ``X = U / ||U||_F``; embeddings, biases and norms keep another
optimiser (:class:`pccl_amd.parallel.Muon`). GPU tensors run the HIP kernels (csrc/hip/hip_muon.hip) on the current
stream without synchronising: every matrix of a call, whatever its shape, goes through each stage in one launch. CPU
tensors run plain torch operations.

A call on the GPU takes a workspace from torch's allocator for its own duration: 8 bytes for each element of X and of
X X^T (sides padded to 64) of every matrix that does not fit in LDS, at most 4 GiB (further matrices take turns in it),
or what one larger matrix needs (20 GiB for 30000 x 60000).
"""
from __future__ import annotations

import ctypes
import math
from functools import lru_cache
from operator import index
from typing import Optional, Sequence, Tuple

import torch

from .._native import C
from ._launch import on_device, refuse_inference, refuse_tangents, require_hip, stream_of
from .kernels import WIRE_DTYPE, _check

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
_TYPES = (torch.float32, torch.bfloat16, torch.float16)


@lru_cache(maxsize=64)
def _check_coefficients(coefficients: Tuple[float, ...], steps: int) -> None:
    """The kernels hold X, A and P = bA + cAA as scaled fp16 pairs (csrc/kernels/muon_common.hpp), so singular values
    have to stay below 4 from the unit interval on, and P's eigenvalues below 12 in size."""
    if len(coefficients) != 3:
        raise ValueError(f"orthogonalize: three coefficients (a, b, c), got {coefficients}")
    if not 1 <= steps <= 100:
        raise ValueError(f"orthogonalize: steps must be in 1..100, got {steps}")
    a, b, c = coefficients
    top = 1.0
    for _ in range(steps):
        s = torch.linspace(0, top, 4097, dtype=torch.float64)
        p = b * s ** 2 + c * s ** 4
        size, nxt = float(p.abs().max()), float((s * (a + p)).abs().max())
        if not (math.isfinite(size) and math.isfinite(nxt)) or size > 11.5 or nxt > 3.9:
            raise ValueError(f"orthogonalize: coefficients {coefficients} let singular values grow out of range")
        top = max(nxt, 1e-30)


def _host_orthogonalize(x: torch.Tensor, steps: int, coefficients, eps: float) -> torch.Tensor:
    a, b, c = coefficients
    norm = x.double().square().sum(dim=(-2, -1), keepdim=True).sqrt()
    y = (x.double() / torch.where(norm < eps, eps, norm)).float()
    flip = y.shape[-2] > y.shape[-1]
    y = y.mT if flip else y
    for _ in range(steps):
        g = y @ y.mT
        y = a * y + (b * g + c * (g @ g)) @ y
    return y.mT if flip else y


def _queue(shapes, g, gtype, w, wtype, mom, alpha, decay, momentum, nesterov, steps, coefficients, eps, device, what):
    """shapes: count, rows, cols of each entry, flat; g, w and mom (None: orthogonalise): addresses."""
    require_hip()
    n = len(g)
    shapes = (ctypes.c_int64 * (3 * n))(*shapes)
    pointers = ctypes.c_void_p * n
    need = C.pcclxMuonWorkspace(n, shapes)
    if need < 0:
        raise ValueError(f"{what}: a matrix is too large")
    with on_device(device):
        work = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        rc = C.pcclxMuon(n, shapes, pointers(*g), WIRE_DTYPE[gtype], pointers(*w), WIRE_DTYPE[wtype],
                         pointers(*mom) if mom else None, (ctypes.c_float * n)(*alpha) if mom else None, decay,
                         momentum, nesterov, steps, _floats(coefficients), eps, work.data_ptr() if need else None, need,
                         stream_of(device))
    if rc == -3:
        raise ValueError(f"{what}: a tensor that is written shares memory with another one of the call")
    _check(rc, what)


@lru_cache(maxsize=64)
def _floats(coefficients: Tuple[float, ...]):
    return (ctypes.c_float * 3)(*coefficients)


def orthogonalize(x: torch.Tensor, *, steps: int = 5, coefficients: Sequence[float] = COEFFICIENTS,
                  eps: float = 1e-7, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The orthogonal factor of each matrix of ``x`` ([..., m, n], fp32 / bf16 / fp16), by ``steps`` Newton-Schulz
    steps from ``x / max(||x||_F, eps)``; singular values end near 1, in about [0.7, 1.2] with the default coefficients.

    Not differentiable (on a GPU a tensor with a forward-mode tangent is refused). The norm is summed in 64 bits; a result
    has the error of fp32 products and one rounding to its type. A zero matrix gives zero, one with a NaN or an infinity gives NaN. Non-contiguous input is copied. ``out`` (contiguous, of x's shape and type) may be ``x`` itself.
    Equal calls give equal bits; a matrix in another stack may differ in its last bits.
    """
    coefficients, steps = tuple(map(float, coefficients)), index(steps)
    _check_coefficients(coefficients, steps)
    if x.dim() < 2:
        raise ValueError(f"orthogonalize: a matrix or a stack of them, got shape {tuple(x.shape)}")
    if x.dtype not in _TYPES:
        raise TypeError(f"orthogonalize: fp32/bf16/fp16, got {x.dtype}")
    if torch.is_grad_enabled() and x.requires_grad:
        raise RuntimeError("orthogonalize is not differentiable: call it under no_grad or on a detached tensor")
    if not eps > 0 or not math.isfinite(eps):
        raise ValueError(f"orthogonalize: eps must be positive, got {eps}")
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    elif out.shape != x.shape or out.dtype != x.dtype or out.device != x.device or not out.is_contiguous():
        raise ValueError("orthogonalize: out must be contiguous and match x in shape, type and device")
    elif torch.is_grad_enabled() and out.requires_grad:
        raise RuntimeError("orthogonalize: out requires a gradient: call it under no_grad")
    refuse_inference("orthogonalize", out)
    if x.numel() == 0:
        return out
    if x.device.type == "cpu":
        return out.copy_(_host_orthogonalize(x, steps, coefficients, eps))
    if x.device.type != "cuda":
        raise ValueError(f"orthogonalize: no kernel for device {x.device}")
    refuse_tangents("orthogonalize", x, out)
    m, n = x.shape[-2:]
    x = x.contiguous()
    _queue((x.numel() // (m * n), m, n), (x.data_ptr(),), x.dtype, (out.data_ptr(),), x.dtype, None, None, 1.0, 0.0, 0,
           steps, coefficients, eps, x.device, "orthogonalize")
    torch.autograd.graph.increment_version(out)
    return out


def _shape_factor(rows: int, cols: int, adjust_lr: str) -> float:
    if adjust_lr == "original":
        return math.sqrt(max(1.0, rows / cols))
    if adjust_lr == "match_rms_adamw":
        return 0.2 * math.sqrt(max(rows, cols))
    if adjust_lr == "none":
        return 1.0
    raise ValueError(f"muon_step: adjust_lr must be 'original', 'match_rms_adamw' or 'none', got {adjust_lr!r}")


def check_muon(what: str, lr: float, weight_decay: float, momentum: float, steps: int,
               coefficients: Sequence[float], eps: float, adjust_lr: str) -> None:
    _check_coefficients(tuple(map(float, coefficients)), steps)
    if not eps > 0 or not math.isfinite(eps):
        raise ValueError(f"{what}: eps must be positive, got {eps}")
    if not 0.0 <= momentum <= 1.0:
        raise ValueError(f"{what}: momentum must be in 0..1, got {momentum}")
    if not (math.isfinite(lr) and math.isfinite(weight_decay)):
        raise ValueError(f"{what}: lr {lr} and weight_decay {weight_decay} must be finite")
    _shape_factor(1, 1, adjust_lr)


def muon_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor],
              momentum_buffers: Sequence[torch.Tensor], *, lr: float, weight_decay: float = 0.1,
              momentum: float = 0.95, nesterov: bool = True, steps: int = 5,
              coefficients: Sequence[float] = COEFFICIENTS, eps: float = 1e-7, adjust_lr: str = "original") -> None:
    """One Muon step on every matrix of ``params``, in place, by torch.optim.Muon's rule:

        buf   = buf + (1 - momentum) (grad - buf)
        u     = grad + momentum (buf - grad) if nesterov else buf
        param = param (1 - lr weight_decay) - lr f(rows, cols) orthogonalize(u)

    with f = sqrt(max(1, rows / cols)) ("original"), 0.2 sqrt(max(rows, cols)) ("match_rms_adamw") or 1 ("none").

    ``params``: contiguous 2-D, one type of fp32 / bf16 / fp16; ``grads``: of their shapes, one type of the same three,
    non-contiguous ones are copied; ``momentum_buffers``: contiguous fp32. All on one device, none of them sharing
    memory with another (a parameter listed twice is refused; a gradient may serve several parameters). Equal calls give
    equal bits on every peer; which matrices share a call decides the order of their sums, so that the same matrix in
    another call may differ in its last bits. The call may be captured into a graph, which then keeps its learning rate.
    """
    coefficients, steps = tuple(map(float, coefficients)), index(steps)
    check_muon("muon_step", lr, weight_decay, momentum, steps, coefficients, eps, adjust_lr)
    if not len(params) == len(grads) == len(momentum_buffers):
        raise ValueError(f"muon_step: {len(params)} parameters, {len(grads)} gradients and {len(momentum_buffers)} "
                         "momentum buffers")
    if not params:
        return
    device, wtype, gtype = params[0].device, params[0].dtype, grads[0].dtype
    if wtype not in _TYPES or gtype not in _TYPES:
        raise TypeError(f"muon_step: fp32/bf16/fp16 parameters and gradients, got {wtype} and {gtype}")
    if device.type not in ("cpu", "cuda"):
        raise ValueError(f"muon_step: no kernel for device {device}")
    work = []
    for p, g, b in zip(params, grads, momentum_buffers):
        shape = p.shape
        if len(shape) != 2 or shape != g.shape or shape != b.shape:
            raise ValueError(f"muon_step: matrices of one shape, got parameter {tuple(shape)}, gradient "
                             f"{tuple(g.shape)}, momentum {tuple(b.shape)}")
        if p.dtype != wtype or g.dtype != gtype:
            raise TypeError("muon_step: parameters, and gradients, must be of one type each")
        if b.dtype != torch.float32:
            raise TypeError(f"muon_step: momentum buffers must be fp32, got {b.dtype}")
        if p.device != device or g.device != device or b.device != device:
            raise ValueError("muon_step: every tensor must be on one device")
        if not p.is_contiguous() or not b.is_contiguous():
            raise ValueError("muon_step: parameters and momentum buffers must be contiguous")
        rows, cols = shape
        if rows and cols:
            work.append((rows, cols, p, g if g.is_contiguous() else g.detach().contiguous(), b))
    if not work:
        return
    refuse_inference("muon_step", *(t for e in work for t in (e[2], e[4])))
    factors = {}
    for e in work:
        if e[:2] not in factors:
            factors[e[:2]] = lr * _shape_factor(*e[:2], adjust_lr)
    alpha = [factors[e[:2]] for e in work]
    decay = 1.0 - lr * weight_decay
    if device.type == "cuda":
        refuse_tangents("muon_step", *(t for e in work for t in e[2:]))
        _queue([v for e in work for v in (1, e[0], e[1])], [e[3].data_ptr() for e in work], gtype,
               [e[2].data_ptr() for e in work], wtype, [e[4].data_ptr() for e in work], alpha, decay, momentum,
               int(nesterov), steps, coefficients, eps, device, "muon_step")
        torch.autograd.graph.increment_version([t for e in work for t in (e[2], e[4])])
        return
    with torch.no_grad():
        end = written_end = 0  # furthest end so far, of any tensor / of the written ones
        for start, stop, written in sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), k > 2)
                                           for e in work for k, t in ((2, e[3]), (3, e[2]), (4, e[4]))):
            if start < written_end or (written and start < end):
                raise ValueError("muon_step: a tensor that is written shares memory with another one of the call")
            end, written_end = max(end, stop), max(written_end, stop if written else 0)
        for (_, _, p, g, b), al in zip(work, alpha):
            g = g.float()
            b.add_(g - b, alpha=1.0 - momentum)
            u = g + momentum * (b - g) if nesterov else b
            p.copy_(p.float() * decay - al * _host_orthogonalize(u, steps, coefficients, eps))
