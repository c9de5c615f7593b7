"""Argument checks and launch plumbing that the policy-training operators share."""

from __future__ import annotations

import contextlib

import torch

from swarp_b200 import _lib

#: torch dtype -> swarp_dtype_t
DTYPES = {torch.float32: 0, torch.float64: 1, torch.bfloat16: 2, torch.float16: 3}

_HERE = contextlib.nullcontext()
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_lib_loaded = None


def library():
    """The loaded library; its checks for a device and a build run on the first call."""
    global _lib_loaded
    if _lib_loaded is None:
        _lib_loaded = _lib.load()
    return _lib_loaded


def stream(device: torch.device) -> int:
    """torch's current stream of ``device``, without a Stream object where torch has a way."""
    return _raw_stream(device.index) if _raw_stream else _lib.stream_ptr(device)


def on_device(device: torch.device):
    """A context in which ``device`` is current: launches go to the current device."""
    return _HERE if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def workspace(nbytes: int, like: torch.Tensor) -> torch.Tensor:
    return like.new_empty(nbytes, dtype=torch.uint8)


def require_cuda(t: torch.Tensor, name: str) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise RuntimeError(f"{name} is on {t.device}: swarp_b200 runs on a CUDA device only "
                           "(no CPU path)")


def like(t: torch.Tensor, name: str, shape, dtypes, device) -> torch.Tensor:
    """``t`` made contiguous, once its shape, dtype and device are what they have to be."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} dtype {t.dtype}: want "
                        f"{' or '.join(str(d) for d in dtypes)}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    return t if t.is_contiguous() else t.contiguous()


def constant(t: torch.Tensor | None, name: str) -> None:
    """Refuse a tensor whose gradient the operator would drop."""
    if t is not None and t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires grad, but no gradient flows to it here: detach it")


__all__ = ["DTYPES", "constant", "library", "like", "on_device", "require_cuda", "stream",
           "workspace"]
