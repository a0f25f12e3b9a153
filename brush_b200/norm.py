"""Group norm with an activation and dropout on channels-last tensors ``[N, ..., C]``, the
layout of the renders (a permuted view of a ``channels_last`` tensor is one without a copy).

Statistics, gates and sums are formed in 32 bits whatever the tensor's type, and rounded once.
Autograd does not record the calls: a result never requires a gradient, and the backward takes the
forward's inputs, statistics and configuration.
"""
from __future__ import annotations

import ctypes as C
import functools
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


@functools.lru_cache(maxsize=1024)
def _sizes(shape: torch.Size, dtype: torch.dtype, param: torch.dtype, groups: int, eps: float, activation: str):
    """(n, pixels, channels, C configuration without dropout, workspace bytes forward, backward) of a call."""
    if len(shape) < 2:
        raise ValueError(f"x must be [N, ..., C], got {tuple(shape)}")
    n, pixels, c = shape[0], math.prod(shape[1:-1]), shape[-1]
    if groups < 1 or c < 1 or c % groups:
        raise ValueError(f"{c} channels cannot be split into {groups} groups")
    if c >= 1 << 32:  # the C interface would see its low half
        raise ValueError("samples x channels must stay below 2^31")
    if pixels == 0:
        raise ValueError("a sample must have at least one pixel")
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}")
    ccfg = _lib.GroupNormCfg(int(groups), float(eps), ACTIVATIONS[activation], DTYPES[param], None)
    need = []
    for backward in (0, 1):
        b = C.c_uint64()
        _lib.check(_lib.lib().bsx_group_norm_workspace(n, pixels, c, groups, backward, C.byref(b)))
        need.append(b.value)
    return n, pixels, c, ccfg, *need


def _call(x: torch.Tensor, weight, bias, cfg: GroupNormConfig):
    """Checks what both directions share: ``_sizes``' values, weight and bias contiguous, and the C configuration."""
    param = None
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor) or t.shape != x.shape[-1:] or t.device != x.device:
            raise ValueError(f"{name} must be a [{x.shape[-1]}] tensor on x's device")
        if param is None:
            param = t.dtype
            if param is not torch.float32 and param is not x.dtype:
                raise ValueError("weight and bias must both be float32 or both of x's type")
        elif t.dtype is not param:
            raise ValueError("weight and bias must both be float32 or both of x's type")
    sizes = _sizes(x.shape, x.dtype, param or torch.float32, cfg.groups, cfg.eps, cfg.activation)
    ccfg = sizes[3]
    if cfg.dropout is not None:
        if cfg.dropout.share != 1:
            raise ValueError("dropout in a group norm draws for each element (share 1)")
        ccfg = _lib.GroupNormCfg(ccfg.groups, ccfg.eps, ccfg.activation, ccfg.param_dtype,
                                 C.pointer(cfg.dropout.to_c(x.device)))
    if weight is not None and not weight.is_contiguous():
        weight = weight.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    return sizes, weight, bias, ccfg


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def _empty(shape: tuple, dtype: torch.dtype, device) -> torch.Tensor:
    """A contiguous [rows, columns] tensor: torch.empty at two thirds of its host time."""
    return torch.empty_strided(shape, (shape[1], 1), dtype=dtype, device=device)


def group_norm_forward(x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None, cfg: GroupNormConfig):
    """(out, mean, rstd): out like x, mean and rstd float [N, groups] for the backward."""
    x = feature_tensor(x, "x")
    (n, pixels, c, _, need, _), weight, bias, ccfg = _call(x, weight, bias, cfg)
    ctx, stream = feature_context(x.get_device())
    out = torch.empty_like(x)
    mean = _empty((n, cfg.groups), torch.float32, x.device)
    rstd = _empty((n, cfg.groups), torch.float32, x.device)
    ws = _empty((need, 1), torch.uint8, x.device) if need else None
    status = _lib.lib().bsx_group_norm_fwd(ctx.handle, x.data_ptr(), _ptr(weight), _ptr(bias), n, pixels, c,
                                           DTYPES[x.dtype], C.byref(ccfg), out.data_ptr(), mean.data_ptr(),
                                           rstd.data_ptr(), _ptr(ws), need, stream)
    if status:
        ctx.check(status)
    return out, mean, rstd


def group_norm_backward(v_output: torch.Tensor, x: torch.Tensor, weight: torch.Tensor | None,
                        bias: torch.Tensor | None, mean: torch.Tensor, rstd: torch.Tensor, cfg: GroupNormConfig):
    """(v_x, v_weight, v_bias) for the forward's inputs, statistics and configuration; the gradient of
    an absent weight or bias is None."""
    x = feature_tensor(x, "x")
    v = like_tensor(v_output, x, "v_output")
    (n, pixels, c, _, _, need), weight, bias, ccfg = _call(x, weight, bias, cfg)
    for t, name in ((mean, "mean"), (rstd, "rstd")):
        if (not isinstance(t, torch.Tensor) or t.shape != (n, cfg.groups) or t.dtype is not torch.float32 or
                t.device != x.device):
            raise ValueError(f"{name} must be the forward's float32 [{n}, {cfg.groups}] tensor")
    mean = mean if mean.is_contiguous() else mean.contiguous()
    rstd = rstd if rstd.is_contiguous() else rstd.contiguous()
    ctx, stream = feature_context(x.get_device())
    v_x = torch.empty_like(x)
    v_weight = None if weight is None else torch.empty_like(weight)
    v_bias = None if bias is None else torch.empty_like(bias)
    ws = _empty((need, 1), torch.uint8, x.device) if need else None
    status = _lib.lib().bsx_group_norm_bwd(ctx.handle, v.data_ptr(), x.data_ptr(), _ptr(weight), _ptr(bias),
                                           mean.data_ptr(), rstd.data_ptr(), n, pixels, c, DTYPES[x.dtype],
                                           C.byref(ccfg), v_x.data_ptr(), _ptr(v_weight), _ptr(v_bias), _ptr(ws), need,
                                           stream)
    if status:
        ctx.check(status)
    return v_x, v_weight, v_bias
