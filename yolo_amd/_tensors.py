"""What every module of the package asks of its tensors: pointers, streams, the current device, and
the checks of arguments."""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd import forward_ad


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _stream(device) -> int:
    """The handle of the current stream of ``device`` (torch.cuda.current_stream builds an object around
    it, which costs several microseconds per call)."""
    index = device.index
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device() if index is None else index)


class _on_device:
    """``torch.cuda.device(dev)`` only when ``dev`` is not already current (the
    context manager costs several microseconds per call otherwise)."""

    __slots__ = ("ctx",)

    def __init__(self, device):
        idx = device.index
        self.ctx = None if idx is None or idx == torch.cuda.current_device() else torch.cuda.device(idx)

    def __enter__(self):
        if self.ctx is not None:
            self.ctx.__enter__()

    def __exit__(self, *exc):
        if self.ctx is not None:
            self.ctx.__exit__(*exc)
        return False


def _tensor(t, name: str, op: str) -> torch.Tensor:
    """A tensor without a forward-mode tangent, which ``op`` would drop."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor, got {type(t).__name__}")
    # the level is -1 outside of forward mode, and asking every tensor costs 0.5 us each
    if getattr(forward_ad, "_current_level", 0) >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"{name}: carries a tangent, and {op} has none; pass its primal part")
    return t


def _forward_only(t, name: str, op: str) -> torch.Tensor:
    """A tensor of which neither a gradient nor a tangent is asked for: ``op`` has none, and would drop it."""
    _tensor(t, name, op)
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name}: requires a gradient, and {op} has none; call it under torch.no_grad() or on a "
                         "detached tensor")
    return t


def _plain(*tensors) -> bool:
    """Whether ``_forward_only`` accepts all of them, asked in one go (0.4 us less for four)."""
    if getattr(forward_ad, "_current_level", 0) >= 0:
        return False
    recorded = torch.is_grad_enabled()
    for t in tensors:
        if t is not None and (not isinstance(t, torch.Tensor) or (recorded and t.requires_grad)):
            return False
    return True


def _need(t: torch.Tensor, name: str, dtype, shape=None) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{name}: must live on the GPU (got device {t.device}); "
                         "yolo_amd has no CPU path")
    if t.dtype != dtype:
        raise ValueError(f"{name}: expected dtype {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: must be contiguous")
    if shape is not None and t.shape != shape and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    return t
