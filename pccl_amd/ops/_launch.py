"""Queueing a kernel on torch's current stream from Python with few host instructions: what the wrappers share."""
from __future__ import annotations

from contextlib import nullcontext

import torch
from torch.autograd import forward_ad

from .kernels import hip_device_count

_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_HERE = nullcontext()


def require_hip() -> None:
    if hip_device_count() == 0:
        raise RuntimeError("pccl-amd HIP backend (libpccl_hip.so) is not loaded but a GPU tensor was passed")


def refuse_tangents(what: str, *tensors: torch.Tensor) -> None:
    """The kernels have no forward-mode derivative, and a dual tensor's tangent would be dropped without a word."""
    if getattr(forward_ad, "_current_level", 0) < 0:  # outside of every dual_level()
        return
    if any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{what}: no forward-mode derivative of the HIP kernels, got a tensor with a tangent")


def refuse_inference(what: str, *written: torch.Tensor) -> None:
    """torch lets nothing write an inference tensor outside of inference mode; asked before anything is written."""
    if any(t.is_inference() for t in written) and not torch.is_inference_mode_enabled():
        raise RuntimeError(f"{what}: an inference tensor would be written outside of inference mode")


def on_device(device: torch.device):
    """A context in which ``device`` is the current one (the kernels are launched on the current device)."""
    return _HERE if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def stream_of(device: torch.device) -> int:
    """The current stream of ``device``; inside :func:`on_device`."""
    return torch.cuda.current_stream(device).cuda_stream if _raw_stream is None else _raw_stream(device.index)
