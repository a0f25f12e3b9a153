"""Dropout with a counter-based mask that is never stored.

``out = residual + x m / (1 - p)``: the mask ``m`` comes from a generator keyed by the seed
and counted by (element, step), as the mean noise of the training step does, so the backward
draws it again instead of reading it, runs are reproducible and ranks with the same seed agree.
``share`` elements in a row use one draw: ``share=1`` drops elements, ``share=C`` drops whole
rows of a ``[N, C]`` tensor (splats, or the rows of a residual branch).

Forward and backward are calls of their own, as everywhere in this package: autograd does not record
them, and a result never requires a gradient (wrap the two in a ``torch.autograd.Function`` for that).
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import torch

from . import _lib
from ._context import feature_context

DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}


@dataclass
class DropoutConfig:
    p: float = 0.1
    seed: int = 42
    # the training step, so that every step draws another mask: an int, or an int32 CUDA tensor of
    # one element that is read when the kernel runs (a captured graph then draws anew at each replay
    # if the tensor changes between replays)
    step: int | torch.Tensor = 0
    share: int = 1

    def to_c(self, device: torch.device) -> _lib.DropoutCfg:
        p, seed, step, share = float(self.p), int(self.seed), self.step, int(self.share)
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"dropout p must lie in [0, 1], got {p}")
        if not 0 <= seed < 1 << 64:
            raise ValueError("dropout seed must be an unsigned 64-bit number")
        if not 1 <= share < 1 << 64:
            raise ValueError("dropout share must be at least 1")
        if isinstance(step, torch.Tensor):
            if step.dtype not in (torch.int32, torch.uint32) or step.numel() != 1 or step.device != device:
                raise ValueError("a dropout step tensor must be one int32 element on the tensor's device")
            return _lib.DropoutCfg(p, seed, share, step.data_ptr(), 0)
        step = int(step)
        if not 0 <= step < 1 << 32:
            raise ValueError("dropout step must be an unsigned 32-bit number")
        return _lib.DropoutCfg(p, seed, share, None, step)


def feature_tensor(t: torch.Tensor, name: str) -> torch.Tensor:
    """``t`` checked for the feature operators, contiguous."""
    if not isinstance(t, torch.Tensor) or t.dtype not in DTYPES:
        raise ValueError(f"{name} must be a float32, bfloat16 or float16 tensor")
    if not t.is_cuda:
        raise ValueError("bsx entry points take CUDA tensors")
    return t if t.is_contiguous() else t.contiguous()


def like_tensor(t: torch.Tensor, x: torch.Tensor, name: str) -> torch.Tensor:
    """``t`` checked to have the shape, type and device of ``x``, contiguous."""
    if not isinstance(t, torch.Tensor) or t.shape != x.shape or t.dtype != x.dtype or t.device != x.device:
        raise ValueError(f"{name} must have the shape, type and device of the tensor it belongs to")
    return t if t.is_contiguous() else t.contiguous()


def dropout_forward(x: torch.Tensor, cfg: DropoutConfig, residual: torch.Tensor | None = None) -> torch.Tensor:
    """``residual + dropout(x)`` in x's shape and type; formed in 32 bits, rounded once."""
    x = feature_tensor(x, "x")
    if residual is not None:
        residual = like_tensor(residual, x, "residual")
    c = cfg.to_c(x.device)
    ctx, stream = feature_context(x.get_device())
    out = torch.empty_like(x)
    status = _lib.lib().bsx_dropout_fwd(ctx.handle, x.data_ptr(), None if residual is None else residual.data_ptr(),
                                        x.numel(), DTYPES[x.dtype], C.byref(c), out.data_ptr(), stream)
    if status:
        ctx.check(status)
    return out


def dropout_backward(v_output: torch.Tensor, cfg: DropoutConfig) -> torch.Tensor:
    """The gradient of x for ``v_output``; the residual's gradient is ``v_output`` itself."""
    v = feature_tensor(v_output, "v_output")
    c = cfg.to_c(v.device)
    ctx, stream = feature_context(v.get_device())
    v_x = torch.empty_like(v)
    status = _lib.lib().bsx_dropout_bwd(ctx.handle, v.data_ptr(), v.numel(), DTYPES[v.dtype], C.byref(c), v_x.data_ptr(),
                                        stream)
    if status:
        ctx.check(status)
    return v_x
