"""Group norm with an activation and dropout on channels-last tensors ``[N, ..., C]``, the
layout of the renders (a permuted view of a ``channels_last`` tensor is one without a copy).

Statistics, gates and sums are formed in 32 bits whatever the tensor's type, and rounded once.
"""
from __future__ import annotations

import ctypes as C
import math
from dataclasses import dataclass

import torch

from . import _lib
from ._context import feature_context
from .dropout import DTYPES, DropoutConfig, feature_tensor, like_tensor

ACTIVATIONS = {"none": _lib.ACT_NONE, "silu": _lib.ACT_SILU, "gelu_tanh": _lib.ACT_GELU_TANH}


@dataclass
class GroupNormConfig:
    groups: int = 32
    eps: float = 1e-5
    activation: str = "none"                # "none", "silu" or "gelu_tanh"
    dropout: DropoutConfig | None = None    # after the activation, share 1


def _call(x: torch.Tensor, weight, bias, cfg: GroupNormConfig):
    """Checks what both directions share: (sizes, C configuration, what the call must keep alive)."""
    if x.dim() < 2:
        raise ValueError(f"x must be [N, ..., C], got {tuple(x.shape)}")
    n, c = x.shape[0], x.shape[-1]
    if cfg.groups < 1 or c < 1 or c % cfg.groups:
        raise ValueError(f"{c} channels cannot be split into {cfg.groups} groups")
    pixels = math.prod(x.shape[1:-1])
    if pixels == 0:
        raise ValueError("a sample must have at least one pixel")
    if not cfg.eps >= 0.0:
        raise ValueError("eps must not be negative")
    if cfg.activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}")
    ptype = None
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor) or t.shape != (c,) or t.device != x.device:
            raise ValueError(f"{name} must be a [{c}] tensor on x's device")
        if t.dtype not in (torch.float32, x.dtype) or t.dtype != (ptype or t.dtype):
            raise ValueError("weight and bias must both be float32 or both of x's type")
        ptype = t.dtype
    drop = None
    if cfg.dropout is not None:
        if cfg.dropout.share != 1:
            raise ValueError("dropout in a group norm draws for each element (share 1)")
        drop = cfg.dropout.to_c(x.device)
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    ccfg = _lib.GroupNormCfg(cfg.groups, cfg.eps, ACTIVATIONS[cfg.activation], DTYPES[ptype or torch.float32],
                             None if drop is None else C.pointer(drop))
    return n, pixels, c, weight, bias, ccfg


def _workspace(n: int, pixels: int, c: int, groups: int, backward: bool, device) -> torch.Tensor:
    need = C.c_uint64()
    _lib.check(_lib.lib().bsx_group_norm_workspace(n, pixels, c, groups, int(backward), C.byref(need)))
    return torch.empty(need.value, dtype=torch.uint8, device=device)


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def group_norm_forward(x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None, cfg: GroupNormConfig):
    """(out, mean, rstd): out like x, mean and rstd float [N, groups] for the backward."""
    x = feature_tensor(x, "x")
    n, pixels, c, weight, bias, ccfg = _call(x, weight, bias, cfg)
    ctx, stream = feature_context(x.device)
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    mean, rstd = torch.empty((2, n, cfg.groups), device=x.device).unbind(0)
    ws = _workspace(n, pixels, c, cfg.groups, False, x.device)
    ctx.check(_lib.lib().bsx_group_norm_fwd(ctx.handle, x.data_ptr(), _ptr(weight), _ptr(bias), n, pixels, c,
                                            DTYPES[x.dtype], C.byref(ccfg), out.data_ptr(), mean.data_ptr(),
                                            rstd.data_ptr(), ws.data_ptr(), ws.numel(), stream))
    return out, mean, rstd


def group_norm_backward(v_output: torch.Tensor, x: torch.Tensor, weight: torch.Tensor | None,
                        bias: torch.Tensor | None, mean: torch.Tensor, rstd: torch.Tensor, cfg: GroupNormConfig):
    """(v_x, v_weight, v_bias) for the forward's inputs, statistics and configuration; the gradient of
    an absent weight or bias is None."""
    x = feature_tensor(x, "x")
    v = like_tensor(v_output, x, "v_output")
    n, pixels, c, weight, bias, ccfg = _call(x, weight, bias, cfg)
    for name, t in (("mean", mean), ("rstd", rstd)):
        if (not isinstance(t, torch.Tensor) or t.shape != (n, cfg.groups) or t.dtype != torch.float32 or
                t.device != x.device):
            raise ValueError(f"{name} must be the forward's float32 [{n}, {cfg.groups}] tensor")
    mean, rstd = mean.contiguous(), rstd.contiguous()
    ctx, stream = feature_context(x.device)
    v_x = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    v_weight = None if weight is None else torch.empty_like(weight)
    v_bias = None if bias is None else torch.empty_like(bias)
    ws = _workspace(n, pixels, c, cfg.groups, True, x.device)
    ctx.check(_lib.lib().bsx_group_norm_bwd(ctx.handle, v.data_ptr(), x.data_ptr(), _ptr(weight), _ptr(bias),
                                            mean.data_ptr(), rstd.data_ptr(), n, pixels, c, DTYPES[x.dtype],
                                            C.byref(ccfg), v_x.data_ptr(), _ptr(v_weight), _ptr(v_bias),
                                            ws.data_ptr(), ws.numel(), stream))
    return v_x, v_weight, v_bias
