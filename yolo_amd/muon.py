"""Orthogonalised updates for weight matrices: ``orthogonalize`` (Newton-Schulz steps towards the nearest
matrix with orthonormal rows), ``muon_step`` (momentum, orthogonalised update and weight step of
matrices of one shape) and ``Muon``, the optimizer made of it, for the convolutions and linear layers in
front of the head (the reference trains them with AdamW, train.py:84-94):

    weights = [p for p in net.parameters() if p.dim() >= 2]
    optim = Muon(weights, lr=0.02)
"""
from __future__ import annotations

import ctypes
import math
from functools import lru_cache
from typing import Optional, Sequence, Tuple

import torch

from . import _lib
from ._tensors import _forward_only, _need, _on_device, _stream, _tensor

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)
# the published coefficients of this update (K. Jordan et al., 2024): they raise small singular values fastest, to 0.7 .. 1.2
COEFFS = (3.4445, -4.7750, 2.0315)


@lru_cache(maxsize=4096)
def _workspace_bytes(count: int, rows: int, cols: int) -> int:
    return _lib.load().yh_orthogonalize_workspace_bytes(count, rows, cols)


def _workspace(count: int, rows: int, cols: int, device) -> torch.Tensor:
    nbytes = _workspace_bytes(count, rows, cols)
    if nbytes == 0:
        raise ValueError(f"{count} matrices of {rows} x {cols}: outside the supported range (at most 65,535 matrices, shorter side "
                         "up to 32,768, longer up to 2^24, and in all fewer than 2^24 tiles of 32 x 32)")
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


_MOST = 3.4028234663852886e38       # of fp32


def _check_steps(steps: int, eps: float) -> None:
    if not 1 <= int(steps) <= _lib.YH_MAX_NS_STEPS:
        raise ValueError(f"steps: expected 1 .. {_lib.YH_MAX_NS_STEPS}, got {steps}")
    if not 0 <= eps <= _MOST:
        raise ValueError(f"eps: expected a finite number that is not negative, got {eps}")


def _check_numbers(coeffs, **numbers) -> None:
    if len(coeffs) != 3:
        raise ValueError(f"coeffs: expected three numbers, got {len(coeffs)}")
    for name, value in (*numbers.items(), *((f"coeffs[{i}]", v) for i, v in enumerate(coeffs))):
        if not abs(value) <= _MOST:
            raise _lib.YoloHeadError(_lib.YH_ERR_ARG, f"{name}: expected a finite number (in fp32), got {value}")


def _check(rc: int) -> None:
    if rc == _lib.YH_ERR_ARG:
        raise _lib.YoloHeadError(rc, "coeffs: coefficients under which so many steps leave the supported range: with singular "
                                     "values s in [0, 1], s^2, |b s^2 + c s^4| or s^2 |a + b s^2 + c s^4| may pass 120 before a step")
    _lib.check(rc)


def orthogonalize(g: torch.Tensor, steps: int = 5, coeffs: Tuple[float, float, float] = COEFFS, eps: float = 1e-7,
                  out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``steps`` times ``X <- (a + b X X' + c (X X')^2) X`` from ``X = g / (|g| + eps)`` for every matrix of
    ``g`` (..., rows, cols), fp32, fp16 or bf16; a matrix taller than wide is worked on transposed.

    Columns lie next to each other and rows at any stride of at least ``cols``; leading axes collapse to one.
    The matrices are held in 22 bits: the result (contiguous, ``out_dtype``) is within about 1e-4 of the exact
    one (whole matrix, relative; 1e-3 when it is bf16) before its rounding, for matrices of up to a few thousand rows.
    Coefficients and steps under which, with singular values s in [0, 1], s^2, |b s^2 + c s^4| or
    s^2 |a + b s^2 + c s^4| may pass 120 before a step are refused.  A NaN or an infinity makes its whole matrix
    NaN.  Forward only."""
    _forward_only(g, "g", "orthogonalize")
    _check_steps(steps, eps)
    _check_numbers(coeffs)
    if not g.is_cuda:
        raise ValueError(f"g: must live on the GPU (got device {g.device}); yolo_amd has no CPU path")
    if g.dtype not in _FLOATS or out_dtype not in _FLOATS:
        raise ValueError(f"g and out_dtype: expected float32, float16 or bfloat16, got {g.dtype} and {out_dtype}")
    if g.dim() < 2:
        raise ValueError(f"g: expected shape (..., rows, cols), got {tuple(g.shape)}")
    out = torch.empty(g.shape, dtype=out_dtype, device=g.device)
    if g.numel() == 0:
        return out
    rows, cols = g.shape[-2:]
    if (cols > 1 and g.stride(-1) != 1) or (rows > 1 and g.stride(-2) < cols):
        raise ValueError("g: columns must lie next to each other and rows at least a row apart (pass g.contiguous(); for a "
                         "transposed matrix orthogonalize the original and transpose the result)")
    batch = g.reshape(-1, rows, cols)
    count = batch.shape[0]
    lib = _lib.load()
    ws = _workspace(count, rows, cols, g.device)
    ld = batch.stride(1) if rows > 1 else cols
    with _on_device(g.device):
        _check(lib.yh_orthogonalize(
            batch.data_ptr(), _lib.DTYPE_CODES[g.dtype], batch.stride(0) if count > 1 else rows * ld, ld, out.data_ptr(),
            _lib.DTYPE_CODES[out_dtype], rows * cols, cols, count, rows, cols, *(float(v) for v in coeffs), int(steps),
            float(eps), ws.data_ptr(), ws.numel(), _stream(g.device)))
    return out


def muon_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], momenta: Sequence[torch.Tensor], lr: float,
              momentum: float = 0.95, weight_decay: float = 0.0, nesterov: bool = True, scale: Optional[float] = None,
              steps: int = 5, coeffs: Tuple[float, float, float] = COEFFS, eps: float = 1e-7) -> None:
    """One step of weights of one shape, in place: ``m <- momentum m + g``; ``u = g + momentum m`` (``nesterov``)
    or ``m``; ``p <- (1 - lr weight_decay) p - lr scale orthogonalize(u)``.

    ``params`` (fp32, fp16 or bf16), ``grads`` (fp32, fp16 or bf16) and ``momenta`` (fp32) are sequences of
    contiguous tensors of one shape each; an axis beyond the second is folded into the columns (a
    convolution's cout x cin*k*k).  ``scale`` defaults to ``sqrt(max(1, rows / cols))``.  A captured graph replays
    the step with the tensors and numbers it was captured with.  Autograd does not record the step."""
    if not (len(params) == len(grads) == len(momenta)):
        raise ValueError(f"{len(params)} params, {len(grads)} grads and {len(momenta)} momenta")
    if not params:
        return
    for name, tensors in (("params", params), ("grads", grads), ("momenta", momenta)):
        for i, t in enumerate(tensors):
            _tensor(t, f"{name}[{i}]", "muon_step")
    _check_steps(steps, eps)
    _check_numbers(coeffs, lr=lr, momentum=momentum, weight_decay=weight_decay, scale=0.0 if scale is None else scale)
    first = params[0]
    shape, dev = tuple(first.shape), first.device
    if len(shape) < 2:
        raise ValueError(f"params: expected at least two axes, got {shape}")
    if first.dtype not in _FLOATS or grads[0].dtype not in _FLOATS:
        raise ValueError(f"params and grads: expected float32, float16 or bfloat16, got {first.dtype} and {grads[0].dtype}")
    for name, tensors, dtype in (("params", params, first.dtype), ("grads", grads, grads[0].dtype),
                                 ("momenta", momenta, torch.float32)):
        for i, t in enumerate(tensors):
            _need(t.detach(), f"{name}[{i}]", dtype, shape)
            if t.device != dev:
                raise ValueError(f"{name}[{i}]: on {t.device}, params[0] is on {dev}")
    if first.numel() == 0:
        return
    spans = sorted([(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), 1) for t in (*params, *momenta)]
                   + [(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), 0) for t in grads])
    end, end_written = 0, 0
    for lo, hi, written in spans:        # what is written overlaps nothing; a gradient may serve two weights
        if lo < end_written or (written and lo < end):
            raise ValueError("params and momenta: each in memory of its own; the same memory is given twice")
        end, end_written = max(end, hi), max(end_written, hi if written else 0)
    rows, cols = shape[0], first.numel() // shape[0]
    if scale is None:
        scale = math.sqrt(max(1.0, rows / cols))
    lib = _lib.load()
    most = _lib.YH_MUON_MAX_COUNT
    for at in range(0, len(params), most):
        some = slice(at, at + most)
        count = len(params[some])
        ws = _workspace(count, rows, cols, dev)
        lists = [(ctypes.c_void_p * count)(*(t.data_ptr() for t in tensors[some])) for tensors in (params, grads, momenta)]
        with _on_device(dev):
            _check(lib.yh_muon_step(
                lists[0], _lib.DTYPE_CODES[first.dtype], lists[1], _lib.DTYPE_CODES[grads[0].dtype], lists[2], count, rows, cols,
                float(lr), float(momentum), int(bool(nesterov)), float(weight_decay), float(scale), *(float(v) for v in coeffs),
                int(steps), float(eps), ws.data_ptr(), ws.numel(), _stream(dev)))
    for t in (*params, *momenta):
        if not t.is_inference():
            torch.autograd.graph.increment_version(t)


class Muon(torch.optim.Optimizer):
    """``muon_step`` as an optimizer over weights of two or more axes (convolutions, linear layers), contiguous or
    channels-last; biases and norms belong to another optimizer.  Weights of one shape, type and layout are stepped together.
    The types and layouts of all weights are looked at before any is changed."""

    def __init__(self, params, lr: float = 0.02, momentum: float = 0.95, weight_decay: float = 0.0, nesterov: bool = True,
                 steps: int = 5, coeffs: Tuple[float, float, float] = COEFFS, eps: float = 1e-7):
        _check_steps(steps, eps)
        super().__init__(params, dict(lr=lr, momentum=momentum, weight_decay=weight_decay, nesterov=nesterov, steps=steps,
                                      coeffs=tuple(coeffs), eps=eps))
        for group in self.param_groups:
            for p in group["params"]:
                if p.dim() < 2:
                    raise ValueError(f"Muon: a parameter of shape {tuple(p.shape)}; weights of two or more axes only")

    def load_state_dict(self, state_dict):
        # torch casts a loaded state to the types of its weights; momenta stay fp32.  They come from what the last
        # pre-hook leaves, and the first post-hook finds them in place.
        loaded = []              # (weight, its momentum)

        def keep(_, given):
            keys = [key for group in given["param_groups"] for key in group["params"]]
            weights = [p for group in self.param_groups for p in group["params"]]
            for key, p in zip(keys, weights):
                saved = given["state"].get(key, {}).get("momentum_buffer")
                if saved is not None:
                    if saved.shape != p.shape:
                        raise ValueError(f"Muon: a momentum of shape {tuple(saved.shape)} for a weight of shape {tuple(p.shape)}")
                    loaded.append((p, saved))

        def restore(_):
            for p, saved in loaded:
                self.state[p]["momentum_buffer"] = torch.empty_like(p, dtype=torch.float32, requires_grad=False).copy_(saved.detach())

        hooks = [self.register_load_state_dict_pre_hook(keep), self.register_load_state_dict_post_hook(restore, prepend=True)]
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        groups, unmade = [], set()
        for group in self.param_groups:               # all of them are looked at before anything is made or changed
            alike = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.dim() < 2:
                    raise ValueError(f"Muon: a parameter of shape {tuple(p.shape)}; weights of two or more axes only")
                if p.dtype not in _FLOATS or p.grad.dtype not in _FLOATS or p.grad.layout != torch.strided:
                    raise ValueError("Muon: expected weights and dense gradients of float32, float16 or bfloat16, got "
                                     f"{p.dtype} and {p.grad.dtype}, {p.grad.layout}")
                order = _rows_outermost(p)
                held = self.state[p].get("momentum_buffer") if p in self.state else None
                if held is None or not _in_order(held, order).is_contiguous():
                    unmade.add(p.device)
                alike.setdefault((tuple(p.shape), p.dtype, p.grad.dtype, p.device, order), []).append(p)
            groups.append((group, alike))
        for dev in unmade:
            with _on_device(dev):
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("Muon: the first step of a weight, or of one that was laid out anew, makes its momentum, and a "
                                       "captured graph would make it in every replay; take one step before the capture")
            if dev.type != "cuda":
                raise ValueError(f"Muon: a parameter on {dev}; yolo_amd has no CPU path")
        for group, alike in groups:
            for (*_, order), ps in alike.items():
                momenta = [self._momentum(p, order) for p in ps]
                muon_step([_in_order(p, order) for p in ps], [_in_order(p.grad, order).contiguous() for p in ps],
                          [_in_order(m, order) for m in momenta], lr=group["lr"], momentum=group["momentum"],
                          weight_decay=group["weight_decay"], nesterov=group["nesterov"], steps=group["steps"],
                          coeffs=group["coeffs"], eps=group["eps"])
        return loss

    def _momentum(self, p: torch.Tensor, order) -> torch.Tensor:
        """The momentum of ``p``, lying as ``p`` does."""
        state = self.state[p]
        held = state.get("momentum_buffer")
        if held is None or not _in_order(held, order).is_contiguous():
            new = torch.zeros_like(p, dtype=torch.float32, requires_grad=False)
            state["momentum_buffer"] = new if held is None else new.copy_(held)
        return state["momentum_buffer"]


def _rows_outermost(p: torch.Tensor) -> Optional[Tuple[int, ...]]:
    """The order of axes, the first one staying first, in which ``p`` is contiguous (None: as they are).  A channels-last
    convolution is a matrix whose columns come in another order, and so do those of its update."""
    if p.is_contiguous():
        return None
    order = (0, *sorted(range(1, p.dim()), key=p.stride, reverse=True))
    if not p.permute(order).is_contiguous():
        raise ValueError(f"Muon: a parameter of shape {tuple(p.shape)} and strides {p.stride()}; its numbers must lie next to each "
                         "other with the first axis outermost (contiguous or channels-last)")
    return order


def _in_order(t: torch.Tensor, order: Optional[Tuple[int, ...]]) -> torch.Tensor:
    return t if order is None else t.permute(order)
