"""Linear layers: the product with bias, activation and residual in its epilogue, and its gradients.

    y = linear(x, w, bias, activation="gelu", residual=r)         # act(x @ w + bias) + r

One launch where x is row-major and w row-major or k-contiguous (``weight.t()``); the tile is the library's built-in choice, no tuning.  Matrices are launched by csrc/launch.cpp;
x of other dimensions is reshaped here and goes through the interpreter, 8 us more a call and some 100 a training step.  For the backward
pass z = x @ w + bias is written beside y where there is an activation.  Gradients: dz = dy * act'(z) and the bias' sums in one pass, then two
products.  Tensors live on a HIP device; there is no CPU path.
"""
from __future__ import annotations

import ctypes
import importlib
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from tritonix_amd import _C
from tritonix_amd import kernel as _kernel
from tritonix_amd.ops import native as _native
from tritonix_amd.ops.mx import as_memory, dtype_code, no_tangent, on_device, raise_for_status

_mm = importlib.import_module("tritonix_amd.ops.matmul")

__all__ = ["linear"]

ACTIVATIONS = {None: _C.ACT_NONE, "relu": _C.ACT_RELU, "silu": _C.ACT_SILU, "gelu": _C.ACT_GELU, "gelu_tanh": _C.ACT_GELU_TANH}


def _go(index: int, x, w, bias, residual, activation: int, want_z: bool):
    m, k = x.shape
    n = w.shape[1]
    if m and n and k:
        x, w, _ = _mm.engine_operands(x, w)
    y = torch.empty((m, n), dtype=x.dtype, device=x.device)
    z = torch.empty_like(y) if want_z else None
    a = _C.LinearArgs()
    a.x, a.w, a.y = x.data_ptr(), w.data_ptr(), y.data_ptr()
    a.bias, a.bias_dtype = (bias.data_ptr(), dtype_code("linear", bias.dtype)) if bias is not None else (None, 0)
    a.residual = residual.data_ptr() if residual is not None else None
    a.z = z.data_ptr() if want_z else None
    a.m, a.n, a.k = m, n, k
    a.stride_xm, a.stride_xk, a.stride_wk, a.stride_wn = *x.stride(), *w.stride()
    a.dtype, a.activation = dtype_code("linear", x.dtype), activation
    lib = _C.load()
    a.stream = stream = _kernel._stream_of(index)
    need, scratch_bytes = int(lib.tnx_linear_workspace_bytes(ctypes.byref(a))), int(lib.tnx_linear_scratch_bytes(ctypes.byref(a)))
    ws = scratch = None
    if need:
        ws = _native.counted_workspace(index, stream, need)
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    if scratch_bytes:
        scratch = torch.empty(scratch_bytes, dtype=torch.uint8, device=x.device)
        a.scratch, a.scratch_bytes = scratch.data_ptr(), scratch_bytes
    status = lib.tnx_linear(ctypes.byref(a))
    if status == _C.E_HIP and need:
        _kernel.drop_workspace(x.device, stream)
    raise_for_status(status, "linear")
    del ws, scratch
    return y, z


def _run(x, w, bias=None, residual=None, activation: int = _C.ACT_NONE, want_z: bool = False):
    """y, and z or None, of matrices on one device."""
    index = x.get_device()
    if index == torch.cuda.current_device():
        return _go(index, x, w, bias, residual, activation, want_z)
    with torch.cuda.device(index):
        return _go(index, x, w, bias, residual, activation, want_z)


def _gradient(dy, z, activation: int, want_dz: bool, bias_dtype):
    """dz (None: not wanted) and the sums of its columns in ``bias_dtype`` (None: not wanted)."""
    m, n = dy.shape
    index = dy.get_device()
    dz = torch.empty_like(dy) if want_dz else None
    dbias = torch.empty(n, dtype=bias_dtype, device=dy.device) if bias_dtype is not None else None
    a = _C.LinearGradientArgs()
    a.dy, a.z = dy.data_ptr(), z.data_ptr() if z is not None else None
    a.dz = dz.data_ptr() if want_dz else None
    a.dbias, a.bias_dtype = (dbias.data_ptr(), dtype_code("linear", bias_dtype)) if dbias is not None else (None, 0)
    a.m, a.n, a.dtype, a.activation = m, n, dtype_code("linear", dy.dtype), activation
    lib = _C.load()
    with torch.cuda.device(index):
        need = int(lib.tnx_linear_gradient_bytes(ctypes.byref(a)))
        scratch = torch.empty(need, dtype=torch.uint8, device=dy.device) if need else None
        if need:
            a.workspace, a.workspace_bytes = scratch.data_ptr(), need
        a.stream = _kernel._stream_of(index)
        raise_for_status(lib.tnx_linear_gradient(ctypes.byref(a)), "linear")
    del scratch
    return dz, dbias


def _transposed(w) -> bool:
    """A k-contiguous w, the transpose of a row-major weight: its gradient gets that layout too."""
    return w.stride(0) == 1 and w.stride(1) != 1


class _Linear(torch.autograd.Function):
    """What the native side has not taken."""

    @staticmethod
    def forward(ctx, x, w, bias, residual, activation):
        derived = activation != _C.ACT_NONE and any(ctx.needs_input_grad[:3])
        y, z = _run(x, w, bias, residual, activation, derived)
        ctx.set_materialize_grads(False)
        # (what no gradient that is asked for reads is not kept: it may change before the backward pass)
        ctx.save_for_backward(x if ctx.needs_input_grad[1] else None, w if ctx.needs_input_grad[0] else None, z)
        ctx.activation, ctx.bias_dtype, ctx.transposed = activation, None if bias is None else bias.dtype, _transposed(w)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        if dy is None:
            return None, None, None, None, None
        no_tangent("linear", dy)
        (dy,) = as_memory(dy)
        x, w, z = ctx.saved_tensors
        wants_x, wants_w, wants_bias, wants_residual = ctx.needs_input_grad[:4]
        dresidual = dy if wants_residual else None
        dx = dw = dbias = None
        if wants_x or wants_w or wants_bias:
            dz = dy = dy.contiguous()
            derived = ctx.activation != _C.ACT_NONE
            if derived or wants_bias:
                made, dbias = _gradient(dy, z, ctx.activation, derived and (wants_x or wants_w), ctx.bias_dtype if wants_bias else None)
                dz = made if derived else dy
            if wants_x:
                dx = _run(dz, w.t())[0]
            if wants_w:
                dw = _run(dz.t(), x)[0].t() if ctx.transposed else _run(x.t(), dz)[0]
        return dx, dw, dbias, dresidual, None


def linear(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: Optional[str] = None,
           residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``act(x @ w + bias) + residual`` with ``x[..., k]``, ``w[k, n]``, ``bias[n]`` and ``residual[..., n]``.

    float16, bfloat16 and float32 (as ``matmul``: three bfloat16 products, off by some 3e-6 of the result's 2-norm, few rows and small problems on the
    binary32 matrix instruction; ``grouped_matmul`` takes that one always); w and residual have x's dtype, the bias that or float32.  ``activation`` is None, "relu", "silu", "gelu" (with erf) or
    "gelu_tanh".  Sums, bias, activation and residual are in 32 bits, the result is rounded once.

    An infinite x @ w + bias has the activation's limits, a NaN stays one.

    Differentiable in x, w, bias and residual, once and backwards: second derivatives and tangents of forward mode are errors.  act' is taken at z = x @ w + bias as it was kept, rounded to x's dtype; dz = dy * act'(z) is
    rounded to it for the products dx = dz @ w.t() and dw = x.t() @ dz, the bias' gradient sums it in 32 bits, in an order that depends on the sizes alone."""
    act = ACTIVATIONS.get(activation)
    if act is not None:
        y = (_native.module or _native.find()).linear(x, w, bias, residual, act)
        if y is not None:
            return y
    else:
        raise ValueError(f"linear: activation is None, 'relu', 'silu', 'gelu' or 'gelu_tanh', got {activation!r}")
    if x.dim() < 1 or w.dim() != 2 or x.shape[-1] != w.shape[0]:
        raise ValueError(f"linear expects x[..., k] and w[k, n], got {tuple(x.shape)} and {tuple(w.shape)}")
    dtype_code("linear", x.dtype)
    if w.dtype != x.dtype or (residual is not None and residual.dtype != x.dtype):
        raise ValueError(f"linear: x is {x.dtype}, w is {w.dtype}" + (f", residual is {residual.dtype}" if residual is not None else ""))
    k, n = w.shape
    if bias is not None and (tuple(bias.shape) != (n,) or bias.dtype not in (x.dtype, torch.float32)):
        raise ValueError(f"linear: bias is [{n}] of {x.dtype} or float32, got {tuple(bias.shape)} of {bias.dtype}")
    lead = tuple(x.shape[:-1])
    if residual is not None and tuple(residual.shape) != (*lead, n):
        raise ValueError(f"linear: residual is {(*lead, n)}, got {tuple(residual.shape)}")
    on_device("linear", x, w, bias, residual)
    rows = 1
    for d in lead:
        rows *= d
    x, w, bias, residual = as_memory(x, w, bias, residual)
    x = x if len(lead) == 1 else x.reshape(rows, k)
    if residual is not None:
        residual = residual.reshape(rows, n).contiguous()
    if bias is not None:
        bias = bias.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        y = _Linear.apply(x, w, bias, residual, act)
    else:
        y = _run(x, w, bias, residual, act)[0]
    return y if len(lead) == 1 else y.reshape(*lead, n)
