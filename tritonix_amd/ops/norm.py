"""Layer normalisation and its gradients.

    y = layer_norm(x, weight, bias)              # (x - mean) / sqrt(variance + eps) * weight + bias over the last dimension

A row is read once (of more than 32768 elements of 16 bits, 16384 of 32, again for each pass); mean, variance and sums are in 32 bits.  The gradients of weight and bias are summed over the rows in an order that depends on the
sizes alone: the same call gives the same bits.  Matrices are launched by csrc/launch.cpp; x of other dimensions is reshaped here and goes through the interpreter, 9 us more a call and some 80 a training step.
Tensors live on a HIP device; there is no CPU path.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from tritonix_amd import _C
from tritonix_amd import kernel as _kernel
from tritonix_amd.ops import native as _native
from tritonix_amd.ops.mx import as_memory, dtype_code, launch, no_tangent, on_device, raise_for_status

__all__ = ["layer_norm"]


def _args(x, weight, bias, eps: float) -> _C.NormArgs:
    a = _C.NormArgs()
    a.x, a.rows, a.n, a.stride_x = x.data_ptr(), x.shape[0], x.shape[1], x.stride(0)
    a.dtype, a.eps = dtype_code("layer_norm", x.dtype), eps
    if weight is not None:
        a.weight, a.weight_dtype = weight.data_ptr(), dtype_code("layer_norm", weight.dtype)
    if bias is not None:
        a.bias, a.bias_dtype = bias.data_ptr(), dtype_code("layer_norm", bias.dtype)
    return a


def _rows(x) -> torch.Tensor:
    """Rows with neighbouring columns, at any pitch."""
    return x if x.stride(1) == 1 or x.shape[1] <= 1 else x.contiguous()


def _forward(x, weight, bias, eps: float, statistics: bool):
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    a = _args(x, weight, bias, eps)
    a.y = y.data_ptr()
    mean = rstd = None
    if statistics:
        mean, rstd = (torch.empty(x.shape[0], dtype=torch.float32, device=x.device) for _ in range(2))
        a.mean, a.rstd = mean.data_ptr(), rstd.data_ptr()
    launch("layer_norm", x.get_device(), _C.load().tnx_layer_norm, a)
    return y, mean, rstd


class _LayerNorm(torch.autograd.Function):
    """What the native side has not taken."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = _forward(x, weight, bias, eps, True)
        ctx.set_materialize_grads(False)
        # (x where dx or dweight is asked for, weight where dx is: what neither reads may change before the backward pass)
        wants_x, wants_weight = ctx.needs_input_grad[:2]
        ctx.save_for_backward(x if wants_x or wants_weight else None, weight if wants_x else None, mean, rstd)
        ctx.weight_dtype, ctx.bias_dtype = (None if t is None else t.dtype for t in (weight, bias))
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        if dy is None:
            return None, None, None, None
        no_tangent("layer_norm", dy)
        (dy,) = as_memory(dy)
        x, weight, mean, rstd = ctx.saved_tensors
        wants_x, wants_weight, wants_bias = ctx.needs_input_grad[:3]
        dy = _rows(dy)
        # (where only the bias asks, dx and dweight are not written and their sums not looked at: dy stands in for x)
        a = _args(dy if x is None else x, weight, None, 0.0)
        a.mean, a.rstd, a.dy, a.stride_dy = mean.data_ptr(), rstd.data_ptr(), dy.data_ptr(), dy.stride(0)
        dx = torch.empty(dy.shape, dtype=dy.dtype, device=dy.device) if wants_x else None
        dweight = torch.empty(dy.shape[1], dtype=ctx.weight_dtype, device=dy.device) if wants_weight else None
        dbias = torch.empty(dy.shape[1], dtype=ctx.bias_dtype, device=dy.device) if wants_bias else None
        if wants_weight:
            a.weight_dtype = dtype_code("layer_norm", ctx.weight_dtype)
        if wants_bias:
            a.bias_dtype = dtype_code("layer_norm", ctx.bias_dtype)
        a.dx, a.dweight, a.dbias = (None if t is None else t.data_ptr() for t in (dx, dweight, dbias))
        lib = _C.load()
        need = int(lib.tnx_layer_norm_workspace_bytes(ctypes.byref(a)))
        index = dy.get_device()
        with torch.cuda.device(index):
            scratch = torch.empty(need, dtype=torch.uint8, device=dy.device) if need else None
            if need:
                a.workspace, a.workspace_bytes = scratch.data_ptr(), need
            a.stream = _kernel._stream_of(index)
            raise_for_status(lib.tnx_layer_norm_backward(ctypes.byref(a)), "layer_norm")
        del scratch
        return dx, dweight, dbias, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(variance + eps) * weight + bias`` over the last dimension of ``x[..., n]`` (float16, bfloat16 or float32), the
    variance being the mean of (x - mean)^2.

    ``weight[n]`` and ``bias[n]``, of x's dtype or float32, may be left out.  The result has x's dtype and shape, rounded once.  A row with a
    NaN or an infinity is NaN.  Differentiable in x, weight and bias, once and backwards."""
    y = (_native.module or _native.find()).layer_norm(x, weight, bias, eps)
    if y is not None:
        return y
    if x.dim() < 1:
        raise ValueError("layer_norm expects x[..., n], got a scalar")
    n = x.shape[-1]
    dtype_code("layer_norm", x.dtype)
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None and (tuple(p.shape) != (n,) or p.dtype not in (x.dtype, torch.float32)):
            raise ValueError(f"layer_norm: {name} is [{n}] of {x.dtype} or float32, got {tuple(p.shape)} of {p.dtype}")
    eps = float(eps)
    if not eps >= 0.0:
        raise ValueError(f"layer_norm: eps is not negative, got {eps}")
    on_device("layer_norm", x, weight, bias)
    rows = 1
    for d in x.shape[:-1]:
        rows *= d
    x, weight, bias = as_memory(x, weight, bias)
    given = x.shape
    x = _rows(x if x.dim() == 2 else x.reshape(rows, n))
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or (bias is not None and bias.requires_grad)):
        y = _LayerNorm.apply(x, weight, bias, eps)
    else:
        y = _forward(x, weight, bias, eps, False)[0]
    return y if len(given) == 2 else y.reshape(given)
