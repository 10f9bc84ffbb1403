"""Products grouped by expert: rows sorted by group, a weight per group, groups of any sizes, with gradients.

    y = grouped_matmul(x, w, routing.offsets)     # y[r] = x[r] @ w[g] for offsets[g] <= r < offsets[g + 1]

What trains the experts that ``moe_route`` or ``moe_plan`` sent the rows to (``routing.order // top_k`` names the tokens in this order).  The groups' bounds
stay on the GPU: nothing waits for them.  Tensors live on a HIP device; there is no CPU path.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from tritonix_amd import _C
from tritonix_amd.ops import native as _native
from tritonix_amd.ops.mx import as_memory, dtype_code, launch, no_tangent, on_device

__all__ = ["grouped_matmul"]


def _row_major(t) -> torch.Tensor:
    """A matrix with neighbouring columns and rows that do not overlap."""
    m, n = t.shape
    if (t.stride(1) == 1 or n <= 1) and (t.stride(0) >= n or m <= 1):
        return t.as_strided((m, n), (t.stride(0) if m > 1 else max(n, 1), 1)) if t.stride() != (n, 1) else t
    return t.contiguous()


def _weights(w) -> torch.Tensor:
    """Matrices that are row-major or k-contiguous, one pitch from each to the next."""
    _, k, n = w.shape
    if (w.stride(2) == 1 and w.stride(1) >= n) or (w.stride(1) == 1 and w.stride(2) >= k):
        return w
    return w.contiguous()


def _padded(t, dim: int) -> torch.Tensor:
    """``t`` with zeros up to a whole 16-byte chunk along ``dim``: rows shorter than a chunk are more than the kernels' loads may read."""
    chunk = 16 // t.element_size()
    more = -t.shape[dim] % chunk
    shape = list(t.shape)
    shape[dim] += more
    out = torch.zeros(shape, dtype=t.dtype, device=t.device)
    out.narrow(dim, 0, t.shape[dim]).copy_(t)
    return out


def _args(form: int, a, b, c, offsets, n: int, k: int, stride_group: int, stride_bk: int, stride_bn: int) -> _C.GroupedArgs:
    g = _C.GroupedArgs()
    g.a, g.b, g.offsets = a.data_ptr(), b.data_ptr(), offsets.data_ptr()
    g.c = c.data_ptr() if c is not None else None
    g.rows, g.n, g.k, g.groups = a.shape[0], n, k, offsets.numel() - 1
    g.stride_ar, g.stride_ak, g.stride_group, g.stride_bk, g.stride_bn = *a.stride(), stride_group, stride_bk, stride_bn
    g.dtype, g.form = dtype_code("grouped_matmul", a.dtype), form
    return g


def _rows_product(x, w, offsets) -> torch.Tensor:
    """Each row times its group's matrix."""
    rows, k = x.shape
    n = w.shape[2]
    if rows == 0 or n == 0 or k == 0:
        return torch.zeros((rows, n), dtype=x.dtype, device=x.device)
    x, w = _row_major(x), _weights(w)
    lib = _C.load()

    def args(c):
        return _args(_C.GROUPED_ROWS, x, w, c, offsets, w.shape[2], k, *w.stride())

    if n < 8 and not lib.tnx_grouped_route(ctypes.byref(args(None)), None):
        w = _padded(w, 2)
    y = torch.empty((rows, w.shape[2]), dtype=x.dtype, device=x.device)
    _launch(args(y), x)
    return y if w.shape[2] == n else y[:, :n].contiguous()


def _weight_gradient(x, dy, offsets) -> torch.Tensor:
    """[groups, k, n]: each group's rows of x, transposed, times its rows of dy."""
    groups, k, n = offsets.numel() - 1, x.shape[1], dy.shape[1]
    if k == 0 or n == 0:
        return torch.zeros((groups, k, n), dtype=x.dtype, device=x.device)
    x, dy = _row_major(x), _row_major(dy)
    lib = _C.load()

    def args(c):
        return _args(_C.GROUPED_WEIGHT_GRADIENT, x, dy, c, offsets, dy.shape[1], x.shape[1], x.shape[1] * dy.shape[1], *dy.stride())

    if min(n, k) < 8 and not lib.tnx_grouped_route(ctypes.byref(args(None)), None):
        x, dy = _padded(x, 1), _padded(dy, 1)
    dw = torch.empty((groups, x.shape[1], dy.shape[1]), dtype=x.dtype, device=x.device)
    _launch(args(dw), x)
    return dw if dw.shape[1:] == (k, n) else dw[:, :k, :n].contiguous()


def _launch(g, device_of) -> None:
    """``tnx_grouped`` with the scratch that it is faster with."""
    need = int(_C.load().tnx_grouped_workspace_bytes(ctypes.byref(g)))
    scratch = torch.empty(need, dtype=torch.uint8, device=device_of.device) if need else None
    if need:
        g.workspace, g.workspace_bytes = scratch.data_ptr(), need
    launch("grouped_matmul", device_of.get_device(), _C.load().tnx_grouped, g)
    del scratch


class _Grouped(torch.autograd.Function):
    """What the native side has not taken."""

    @staticmethod
    def forward(ctx, x, w, offsets):
        ctx.set_materialize_grads(False)
        # (what no gradient that is asked for reads is not kept: it may change before the backward pass)
        ctx.save_for_backward(x if ctx.needs_input_grad[1] else None, w if ctx.needs_input_grad[0] else None, offsets)
        ctx.transposed = w.stride(1) == 1 and w.stride(2) != 1
        return _rows_product(x, w, offsets)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        if dy is None:
            return None, None, None
        no_tangent("grouped_matmul", dy)
        (dy,) = as_memory(dy)
        x, w, offsets = ctx.saved_tensors
        dx = dw = None
        if ctx.needs_input_grad[0]:
            dx = _rows_product(dy, w.transpose(1, 2), offsets)
        if ctx.needs_input_grad[1]:
            # (a transposed weight's gradient has its layout)
            dw = _weight_gradient(dy, x, offsets).transpose(1, 2) if ctx.transposed else _weight_gradient(x, dy, offsets)
        return dx, dw, None


def grouped_matmul(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """``y[r] = x[r] @ w[g]`` for the rows ``offsets[g] <= r < offsets[g + 1]`` of each group: ``x[rows, k]``, ``w[groups, k, n]``, ``y[rows, n]``.

    float16, bfloat16 and float32 (on the binary32 matrix instruction, at a third of the rate of ``linear``'s three bfloat16 products and exact to 32 bits); sums in 32 bits, rounded once.  ``offsets[groups + 1]`` (int32, or int64) does
    not decrease and lies in ``[0, rows]``; what does not is taken into that.  Groups may be empty; rows of none, ahead of ``offsets[0]`` and from
    ``offsets[groups]`` on, are zero.  w may be the transpose of row-major ``[groups, n, k]`` weights.

    Differentiable in x and w, once and backwards: rows of no group have zero gradients, and so has the weight of a group without rows."""
    y = (_native.module or _native.find()).grouped_matmul(x, w, offsets)
    if y is not None:
        return y
    if x.dim() != 2 or w.dim() != 3 or x.shape[1] != w.shape[1]:
        raise ValueError(f"grouped_matmul expects x[rows, k] and w[groups, k, n], got {tuple(x.shape)} and {tuple(w.shape)}")
    groups = w.shape[0]
    if not 1 <= groups <= _C.GROUPED_MAX_GROUPS:
        raise ValueError(f"grouped_matmul: {groups} groups (1 to {_C.GROUPED_MAX_GROUPS} are built)")
    if tuple(offsets.shape) != (groups + 1,) or offsets.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"grouped_matmul: offsets are int32 or int64 [{groups + 1}], got {offsets.dtype} {tuple(offsets.shape)}")
    dtype_code("grouped_matmul", x.dtype)
    if w.dtype != x.dtype:
        raise ValueError(f"grouped_matmul: x is {x.dtype}, w is {w.dtype}")
    on_device("grouped_matmul", x, w, offsets)
    x, w, offsets = as_memory(x, w, offsets)
    if offsets.dtype == torch.int64:
        offsets = offsets.clamp(0, x.shape[0])             # (past 32 bits: the nearest inside)
    offsets = offsets.to(torch.int32).contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad):
        return _Grouped.apply(x, w, offsets)
    return _rows_product(x, w, offsets)
