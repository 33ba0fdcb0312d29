"""The product of a linear layer in 8-bit integers, for serving the layers in front of the
head (model.py:133-135): ``y = s_m t_n sum_k q_mk w_nk + bias_n`` with a scale for every row of
the input (an image's features) and of the weight (an output channel).

    layer = Int8Linear.from_linear(net[-1])               # weights quantised and laid out once
    dets, count = head.postprocess_linear(features, layer)

The sum is exact in int32; scales and bias are applied in fp32.  Forward only: an input, scale or bias that
requires a gradient while gradients are recorded is refused."""
from __future__ import annotations

from functools import lru_cache
from typing import Optional

import torch
from torch import nn

from . import _lib
from ._tensors import _forward_only, _need, _on_device, _plain, _ptr, _stream

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


@lru_cache(maxsize=4096)
def _workspace_bytes(code: int, m: int, n: int, k: int) -> int:
    return _lib.load().yh_linear_i8_workspace_bytes(code, m, n, k)


def _rows(x: torch.Tensor, name: str) -> torch.Tensor:
    """(..., K) as (M, K) with unit stride along K; a view where the strides allow one."""
    if not x.is_cuda:
        raise ValueError(f"{name}: must live on the GPU (got device {x.device}); yolo_amd has no CPU path")
    shape = x.shape
    if not shape or not 1 <= shape[-1] <= _lib.YH_MAX_I8_K:
        raise ValueError(f"{name}: expected shape (..., K) with K in 1 .. {_lib.YH_MAX_I8_K}, got {tuple(shape)}")
    k = shape[-1]
    if k > 1 and x.stride(-1) != 1:
        raise ValueError(f"{name}: must be contiguous along its last axis")
    m = shape[0] if len(shape) == 2 else x.numel() // k
    if m > _lib.YH_MAX_I8_ROWS:
        raise ValueError(f"{name}: expected at most {_lib.YH_MAX_I8_ROWS:,} rows, got shape {tuple(shape)}")
    if x.requires_grad:
        x = x.detach()
    if len(shape) != 2:
        x = x.reshape(-1, k) if m else x.new_empty(0, k)
    if m > 1 and x.stride(0) < k:                        # expanded or overlapping rows
        x = x.contiguous()
    return x


def _ld(x: torch.Tensor) -> int:
    return x.stride(0) if x.shape[0] > 1 else max(x.stride(0), x.shape[1])


def quantize_rows(x: torch.Tensor):
    """``x`` (M, K) fp32, fp16 or bf16 -> ``(q, scale)``: ``scale[m] = max_k |x[m, k]| / 127`` (fp32) and
    ``q[m, k] = 127 x[m, k] / max_k |x[m, k]|`` to the nearest whole number, ties to even, as int8.

    ``q`` has shape (M, K); its rows lie a multiple of 128 bytes apart with zeros behind them, the
    layout ``linear_i8`` takes for a weight.  A row of zeros gets scale 0; a row that holds a NaN or
    an infinity gets scale NaN and zeros."""
    _forward_only(x, "x", "quantize_rows")
    if x.dim() != 2:
        raise ValueError(f"x: expected shape (M, K), got {tuple(x.shape)}")
    x = _rows(x, "x")
    if x.dtype not in _FLOATS:
        raise ValueError(f"x: expected dtype float32, float16 or bfloat16, got {x.dtype}")
    m, k = x.shape
    q = torch.empty(m, (k + 127) // 128 * 128, dtype=torch.int8, device=x.device)
    scale = torch.empty(m, dtype=torch.float32, device=x.device)
    with _on_device(x.device):
        _lib.check(_lib.load().yh_quantize_rows(x.data_ptr(), _lib.DTYPE_CODES[x.dtype], _ld(x), q.data_ptr(), q.shape[1],
                                                scale.data_ptr(), m, k, _stream(x.device)))
    return q[:, :k], scale


def linear_i8(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
              x_scale: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``y[..., n] = s t_n sum_k q_k w_nk + bias_n``: ``x`` (..., K) times ``weight`` (N, K) int8 with ``weight_scale`` (N).

    ``x`` is fp32, fp16 or bf16 and is quantised row by row as ``quantize_rows`` does, or int8 with the
    scales of its rows in ``x_scale``.  ``weight`` as ``quantize_rows`` returns it: unit stride along K, rows a
    multiple of 16 bytes apart.  ``bias`` (N) fp32.  The result has ``out_dtype`` (fp32, fp16, bf16; by
    default that of ``x``, fp32 for an int8 ``x``)."""
    if x is None or not _plain(x, weight_scale, bias, x_scale):
        for name, t in (("x", x), ("weight_scale", weight_scale), ("bias", bias), ("x_scale", x_scale)):
            if t is not None or name == "x":
                _forward_only(t, name, "linear_i8")
    shape = x.shape
    x = _rows(x, "x")
    m, k = x.shape
    dev = x.device
    code = _lib.DTYPE_CODES.get(x.dtype)
    if code is None:
        raise ValueError(f"x: expected dtype float32, float16, bfloat16 or int8, got {x.dtype}")
    if (code == _lib.YH_I8) != (x_scale is not None):
        raise ValueError("x_scale: the scales of an int8 x, and of nothing else")
    if x_scale is not None:
        _need(x_scale, "x_scale", torch.float32)
        if x_scale.numel() != m:
            raise ValueError(f"x_scale: expected {m} values, got {x_scale.numel()}")
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or weight.shape[1] != k or weight.dtype != torch.int8:
        raise ValueError(f"weight: expected an int8 tensor of shape (N, {k})")
    n = weight.shape[0]
    if n > _lib.YH_MAX_I8_ROWS or (m + 31) // 32 * ((n + 31) // 32) >= 1 << 24:
        raise ValueError(f"weight: expected at most {_lib.YH_MAX_I8_ROWS:,} rows, and a result of fewer than 2^24 tiles of 32 x 32; got "
                         f"{m} x {n}")
    room = (k + 15) // 16 * 16
    ldw, along = weight.stride()
    ldw = ldw if n > 1 else room
    if n and ((along != 1 and k > 1) or ldw < k or ldw % 16 or weight.data_ptr() % 16
              or weight.storage_offset() + (n - 1) * ldw + room > weight.untyped_storage().nbytes()):
        raise ValueError("weight: unit stride along K, rows a multiple of 16 bytes apart and 16-byte aligned, the last one "
                         "with room up to the next multiple of 16 bytes (quantize_rows lays it out so)")
    _need(weight_scale, "weight_scale", torch.float32, (n,))
    if bias is not None:
        _need(bias, "bias", torch.float32, (n,))
    if (weight.device != dev or weight_scale.device != dev or (bias is not None and bias.device != dev)
            or (x_scale is not None and x_scale.device != dev)):
        places = {name: t.device for name, t in (("weight", weight), ("weight_scale", weight_scale), ("bias", bias),
                                                 ("x_scale", x_scale)) if t is not None and t.device != dev}
        raise ValueError(f"{', '.join(places)}: on {', '.join(map(str, places.values()))}, x is on {dev}")
    if out_dtype is None:
        out_dtype = torch.float32 if code == _lib.YH_I8 else x.dtype
    if out_dtype not in _FLOATS:
        raise ValueError(f"out_dtype: expected float32, float16 or bfloat16, got {out_dtype}")
    y = torch.empty((*shape[:-1], n), dtype=out_dtype, device=dev)
    if m == 0 or n == 0:
        return y
    nbytes = _workspace_bytes(code, m, n, k)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    with _on_device(dev):
        _lib.check(_lib.load().yh_linear_i8(
            x.data_ptr(), code, _ld(x), _ptr(x_scale), weight.data_ptr(), ldw, weight_scale.data_ptr(), _ptr(bias),
            y.data_ptr(), _lib.DTYPE_CODES[out_dtype], n, m, n, k, _ptr(ws), nbytes, _stream(dev)))
    return y


class Int8Linear(nn.Module):
    """A linear layer served in 8-bit integers: ``forward(x)`` is ``linear_i8`` with this layer's weight,
    scales and bias.  The weight is quantised and laid out once, by ``from_linear``; weight, scales and bias keep
    their types when the network around them is moved to another (``half()``, ``to(dtype)``)."""

    def __init__(self, weight: torch.Tensor, weight_scale: torch.Tensor, bias: Optional[torch.Tensor] = None):
        super().__init__()
        self.out_features, self.in_features = weight.shape
        rows = weight.new_zeros(self.out_features, (self.in_features + 127) // 128 * 128)
        rows[:, :self.in_features] = weight
        self.register_buffer("weight_rows", rows)
        self.register_buffer("weight_scale", weight_scale.detach().clone())
        self.register_buffer("bias", None if bias is None else bias.detach().float().clone())

    def _apply(self, fn, recurse=True):
        # A network moved to another number type takes the layer along, but the layer keeps its own types: integers for the
        # weight, fp32 for scales and bias.
        held = dict(self._buffers)
        super()._apply(fn, recurse)
        for name, old in held.items():
            if old is not None and self._buffers[name].dtype != old.dtype:
                self._buffers[name] = old.to(self._buffers[name].device)
        return self

    @classmethod
    def from_linear(cls, linear: nn.Linear) -> "Int8Linear":
        """The weight of ``linear`` (fp32, fp16 or bf16, on the GPU) with a scale for each output channel."""
        with torch.no_grad():
            q, scale = quantize_rows(linear.weight.detach().contiguous())
            return cls(q, scale, linear.bias)

    @property
    def weight(self) -> torch.Tensor:
        """(out_features, in_features) int8, rows a multiple of 128 bytes apart."""
        return self.weight_rows[:, :self.in_features]

    def forward(self, x: torch.Tensor, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        return linear_i8(x, self.weight, self.weight_scale, bias=self.bias, out_dtype=out_dtype)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"
