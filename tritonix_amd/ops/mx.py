"""Microscaled 4-bit floats: quantisation, products, the gated product and a linear layer's training step.

An element is a 4-bit float (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign), 32 neighbours along the quantised dimension share a
power-of-two scale held in a byte: 17 bits for four elements, and the type gfx950's matrix cores are fastest in.  A product
contracts along the dimension that both operands are quantised along, so a matrix that enters two products along different dimensions
(the activations of a training step) is quantised twice.

``mx_quantize(x, dim)`` -> ``MXTensor``; ``mx_matmul(a, b)`` is ``a @ b`` with ``a[m, k]`` quantised along its last
dimension and ``b[k, n]`` along its first; a torch tensor in place of either is quantised on the way in.  ``mx_glu`` is ``glu`` of
such operands.  ``mx_linear`` is differentiable: the gradient passes the rounding as if it were not there, and the gradients' products are
microscaled as well.  Tensors live on a HIP device; there is no CPU path.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from tritonix_amd import _C
from tritonix_amd.kernel import _stream_of, launch_module

__all__ = ["MXTensor", "mx_quantize", "mx_dequantize", "mx_matmul", "mx_glu", "mx_linear"]

BLOCK = 32
SLAB = 256                      # k is padded to whole slabs (csrc/mx.h)
# Rows that moe_down joins are in 32 bits, in float16 whatever their number: a row may lie past 65504 where the weighted sum does not (8192 tokens of 8
# experts, 1024 to 4096: 686 us, rounded to 16 bits 460).  bfloat16 has the range: its rows are in 32 bits up to this many bytes, which the L2 caches hold
# together; more of them, whose writing and reading is what the join costs (1 GB each way in 32 bits: 467 us instead of 690), are rounded first.  With eight
# experts that takes the result's error, relative to the exact sum, from 0.0017 to 0.0024 (root mean square; the result's own rounding is the first).
JOIN_BYTES = 32 << 20
_DTYPES = {torch.float16: _C.F16, torch.bfloat16: _C.BF16, torch.float32: _C.F32}
_EPILOGUES = {"silu": _C.EPI_GLU_SILU, "sigmoid": _C.EPI_GLU_SIGMOID}


class _Interpreter:
    """Stands in for ``_launch`` where it cannot be used: every call takes the ordinary path below."""

    @staticmethod
    def _none(*_):
        return None

    mx_quantize = mx_dequantize = mx_product = mx_linear = moe_route = moe_backward = _none


# csrc/launch.cpp, which makes the ordinary calls without the interpreter's share of them; found with the first call
native = None


def find_native():
    global native
    module = launch_module()
    if module is None:
        native = _Interpreter
    else:
        lib = _C.load()
        module.bind_ops(tuple(ctypes.cast(fn, ctypes.c_void_p).value for fn in (
            lib.tnx_mx_code_bytes, lib.tnx_mx_scale_bytes, lib.tnx_mx_quantize, lib.tnx_mx_quantize_both, lib.tnx_mx_dequantize, lib.tnx_mx_gemm_takes_rows, lib.tnx_mx_gemm, lib.tnx_mx_gemm_workspace_bytes,
            lib.tnx_moe_workspace_bytes, lib.tnx_moe_route, lib.tnx_moe_route_backward, lib.tnx_moe_combine)) + (JOIN_BYTES,))
        native = module
    return native


def dtype_code(name: str, dtype) -> int:
    code = _DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"{name}: dtype {dtype} has no HIP kernel (float16, bfloat16 and float32 are built)")
    return code


def raise_for_status(status: int, what: str) -> None:
    if status == _C.OK:
        return
    if status == _C.E_HIP:
        raise RuntimeError(f"{what}: {_C.strerror(status)} (hipError_t {_C.load().tnx_last_hip_error()})")
    if status == _C.E_WORKSPACE:
        raise RuntimeError(f"{what}: {_C.strerror(status)}")
    raise ValueError(f"{what}: {_C.strerror(status)}")


def on_device(name: str, *tensors) -> int:
    """Index of the HIP device that all of them are on."""
    index = -1
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError(f"{name}: tensors must be on a HIP device (there is no CPU path)")
        here = t.get_device()
        if index >= 0 and here != index:
            raise ValueError(f"{name}: tensors are on different devices")
        index = here
    return index


def launch(what: str, index: int, fn, args) -> None:
    """``fn(args)`` on torch's current stream of the device."""
    if index == torch.cuda.current_device():
        args.stream = _stream_of(index)
        status = fn(ctypes.byref(args))
    else:
        with torch.cuda.device(index):
            args.stream = _stream_of(index)
            status = fn(ctypes.byref(args))
    if status:
        raise_for_status(status, what)


class _Underived(torch.autograd.Function):
    """``out`` as it is, with a place in the graph of its inputs: an error where a gradient is asked to pass."""

    @staticmethod
    def forward(ctx, name, out, *inputs):
        ctx.name = name
        return out[0]                                      # (in a list: not an input itself)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError(f"{ctx.name} passes no gradient to its inputs; detach them, or the result, where none is wanted (mx_linear has one)")


def underived(name: str, out: torch.Tensor, *inputs) -> torch.Tensor:
    """The result of an operator without a derivative.  Differentiating it is an error where an input asks for its gradient: left out of the graph, the
    input's gradient would lack this term silently."""
    for t in inputs:
        if t.requires_grad and torch.is_grad_enabled():
            return _Underived.apply(name, [out], *(i for i in inputs if i.requires_grad))
    return out


class MXTensor:
    """A matrix, or a batch of them, in microscaled 4-bit floats.

    ``dim`` is the quantised dimension, -1 or -2; ``shape`` the logical shape.  The memory is the same either way -- rows
    along the quantised dimension -- so ``t()`` costs nothing.  ``codes`` and ``scales`` are the two buffers as the
    kernels read them (include/tritonix_hip.h)."""

    __slots__ = ("buffer", "batch", "rows", "k", "dim", "code_bytes")
    requires_grad = False

    def __init__(self, buffer: torch.Tensor, batch: Optional[int], rows: int, k: int, dim: int, code_bytes: int):
        self.buffer, self.batch, self.rows, self.k, self.dim, self.code_bytes = buffer, batch, rows, k, dim, code_bytes

    @staticmethod
    def empty(batch: Optional[int], rows: int, k: int, dim: int, device) -> "MXTensor":
        slabs = -(-k // SLAB)
        count = 1 if batch is None else batch
        code_bytes = count * rows * slabs * (SLAB // 2)
        scale_bytes = count * (-(-rows // 32)) * (-(-slabs // 2)) * 32 * 2 * (SLAB // BLOCK)
        return MXTensor(torch.empty(code_bytes + scale_bytes, dtype=torch.uint8, device=device), batch, rows, k, dim, code_bytes)

    @staticmethod
    def from_codes(codes: torch.Tensor, scales: torch.Tensor, k: int, dim: int = -1) -> "MXTensor":
        """From the form of checkpoints: ``codes[..., rows, ceil(k / 2)]`` (two a byte, the even element low) and
        ``scales[..., rows, ceil(k / 32)]`` (exponent + 127), uint8, quantised along ``k``.  ``dim=-1`` gives a tensor of shape
        ``[..., rows, k]``, ``dim=-2`` its transpose ``[..., k, rows]``, the right operand of a product; from 0 on it counts the dimensions of that
        shape, as in ``mx_quantize``.  The data is copied."""
        dim = _dim("MXTensor.from_codes", dim, max(codes.dim(), 2))
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise ValueError("MXTensor.from_codes: codes and scales are uint8")
        if codes.dim() not in (2, 3) or k < 1 or codes.shape[-1] != -(-k // 2) or tuple(scales.shape) != (*codes.shape[:-1], -(-k // BLOCK)):
            raise ValueError(f"MXTensor.from_codes: codes {tuple(codes.shape)} and scales {tuple(scales.shape)} are not "
                             f"[..., rows, {-(-k // 2)}] and [..., rows, {-(-k // BLOCK)}]")
        index = on_device("MXTensor.from_codes", codes, scales)
        batch, rows = (codes.shape[0] if codes.dim() == 3 else None), codes.shape[-2]
        out = MXTensor.empty(batch, rows, k, dim, codes.device)
        codes, scales = codes.contiguous(), scales.contiguous()
        with torch.cuda.device(index):
            status = _C.load().tnx_mx_import(codes.data_ptr(), scales.data_ptr(), 1 if batch is None else batch, rows, k, out.codes_ptr,
                                             out.scales_ptr, _stream_of(index))
        raise_for_status(status, "MXTensor.from_codes")
        return out

    @property
    def codes_ptr(self) -> int:
        return self.buffer.data_ptr()

    @property
    def scales_ptr(self) -> int:
        return self.buffer.data_ptr() + self.code_bytes

    @property
    def codes(self) -> torch.Tensor:
        return self.buffer[:self.code_bytes]

    @property
    def scales(self) -> torch.Tensor:
        return self.buffer[self.code_bytes:]

    @property
    def shape(self) -> Tuple[int, ...]:
        matrix = (self.rows, self.k) if self.dim == -1 else (self.k, self.rows)
        return matrix if self.batch is None else (self.batch, *matrix)

    @property
    def device(self):
        return self.buffer.device

    @property
    def is_cuda(self) -> bool:
        return self.buffer.is_cuda

    def get_device(self) -> int:
        return self.buffer.get_device()

    def t(self) -> "MXTensor":
        return MXTensor(self.buffer, self.batch, self.rows, self.k, -3 - self.dim, self.code_bytes)

    def __repr__(self):
        return f"MXTensor(shape={self.shape}, dim={self.dim}, device={self.device})"


def _dim(name: str, dim: int, ndim: int = 2) -> int:
    if dim in (-1, ndim - 1):
        return -1
    if dim in (-2, ndim - 2):
        return -2
    raise ValueError(f"{name}: dim {dim} is not one of the matrix's two")


def _mx_args(data: torch.Tensor, t: MXTensor, code: int) -> _C.MxArgs:
    a = _C.MxArgs()
    a.data, a.codes, a.scales = data.data_ptr(), t.codes_ptr, t.scales_ptr
    a.batch, a.rows, a.k = 1 if t.batch is None else t.batch, t.rows, t.k
    a.stride_batch = 0 if t.batch is None else data.stride(0)
    outer, inner = data.stride(-2), data.stride(-1)
    a.stride_row, a.stride_k = (outer, inner) if t.dim == -1 else (inner, outer)
    a.dtype = code
    return a


def mx_quantize(x: torch.Tensor, dim: int = -1) -> MXTensor:
    """``x`` (float16, bfloat16 or float32, a matrix or a batch of them, any strides) with blocks of 32 along ``dim``.

    A block's scale is 2^(floor(log2 of its largest magnitude) - 2); elements round to the nearest 4-bit float, ties to
    the even code, and those past 6 scales to 6.  A block with an infinity or a NaN becomes NaN throughout.  An ``MXTensor`` is data: it has no place in
    the autograd graph."""
    if dim in (0, 1, -1, -2):
        last = dim in (1, -1)
        got = (native or find_native()).mx_quantize(x, last)             # (a matrix of the current device)
        if got is not None:
            m, n = x.shape
            return MXTensor(got[0], None, m if last else n, n if last else m, -1 if last else -2, got[1])
    if x.dim() not in (2, 3):
        raise ValueError(f"mx_quantize expects a matrix or a batch of them, got {tuple(x.shape)}")
    dim = _dim("mx_quantize", dim, x.dim())
    code = dtype_code("mx_quantize", x.dtype)
    index = on_device("mx_quantize", x)
    rows, k = (x.shape[-2], x.shape[-1]) if dim == -1 else (x.shape[-1], x.shape[-2])
    t = MXTensor.empty(x.shape[0] if x.dim() == 3 else None, rows, k, dim, x.device)
    launch("mx_quantize", index, _C.load().tnx_mx_quantize, _mx_args(x, t, code))
    return t


def mx_dequantize(t: MXTensor, dtype=torch.bfloat16) -> torch.Tensor:
    """The values that ``t`` stands for, contiguous in its logical shape.  (Exact in bfloat16 and float32.)"""
    code = dtype_code("mx_dequantize", dtype)
    if t.batch is None:
        out = (native or find_native()).mx_dequantize(t.buffer, t.code_bytes, t.rows, t.k, int(t.dim == -1), code)
        if out is not None:
            return out
    index = on_device("mx_dequantize", t)
    out = torch.empty(t.shape, dtype=dtype, device=t.device)
    launch("mx_dequantize", index, _C.load().tnx_mx_dequantize, _mx_args(out, t, code))
    return out


def operand(name: str, side: str, x, dim: int) -> MXTensor:
    """``x`` as a microscaled operand that is quantised along ``dim``."""
    if isinstance(x, MXTensor):
        if x.dim != dim:
            raise ValueError(f"{name}: {side} of shape {x.shape} has to be quantised along the dimension that is summed over")
        return x
    return mx_quantize(x, dim=dim)


def takes_rows(x) -> bool:
    """Whether a product takes these rows as they are: a few rows of floats are quantised by the kernel itself."""
    return (not isinstance(x, MXTensor) and 0 < x.shape[0] <= 16 and (x.stride(1) == 1 or x.shape[1] == 1) and x.dtype in _DTYPES
            and bool(_C.load().tnx_mx_gemm_takes_rows(x.shape[0], x.shape[1])))


def gemm_args(a, b: MXTensor, out: torch.Tensor, epilogue: int) -> _C.MxGemmArgs:
    g = _C.MxGemmArgs()
    if isinstance(a, MXTensor):
        g.a_codes, g.a_scales, g.a_rows = a.codes_ptr, a.scales_ptr, a.rows
    else:
        g.a_data, g.a_dtype, g.stride_a, g.a_rows = a.data_ptr(), _DTYPES[a.dtype], a.stride(0), a.shape[0]
    g.b_codes, g.b_scales = b.codes_ptr, b.scales_ptr
    g.out = out.data_ptr()
    g.m, g.n, g.k = out.shape[0], b.rows, b.k
    g.stride_out = out.stride(0)
    g.out_dtype, g.epilogue = _DTYPES[out.dtype], epilogue
    return g


def _product(name: str, a, b, out_dtype, epilogue: int) -> torch.Tensor:
    given = b
    if type(b) is not MXTensor and not isinstance(a, MXTensor) and len(a.shape) == len(b.shape) == 2 and a.shape[1] == b.shape[0]:
        b = mx_quantize(b, dim=0)
    if type(b) is MXTensor and b.batch is None and b.dim == -2 and (out_dtype is None or out_dtype is getattr(a, "dtype", None)):
        out = (native or find_native()).mx_product(a, b.buffer, b.code_bytes, b.rows, b.k, epilogue)
        if out is not None:
            return out if given is b and not a.requires_grad else underived(name, out, a, given)
    if len(a.shape) != 2 or len(b.shape) != 2 or a.shape[1] != b.shape[0]:
        raise ValueError(f"{name} expects a[m,k] and b[k,n], got {tuple(a.shape)} and {tuple(b.shape)}")
    if out_dtype is None:
        out_dtype = torch.bfloat16 if isinstance(a, MXTensor) else a.dtype
    dtype_code(name, out_dtype)
    index = on_device(name, a, b)
    m, k = a.shape
    inputs = (a, given)
    if not takes_rows(a):
        a = operand(name, "a", a, -1)
    b = operand(name, "b", b, -2)
    n = b.rows
    if epilogue != _C.EPI_NONE:
        if n % 2:
            raise ValueError("the interleaved weight must have an even number of columns")
        n //= 2
    if k == 0:
        return underived(name, torch.zeros((m, n), dtype=out_dtype, device=b.device), *inputs)
    out = torch.empty((m, n), dtype=out_dtype, device=b.device)
    g = gemm_args(a, b, out, epilogue)
    nbytes = int(_C.load().tnx_mx_gemm_workspace_bytes(ctypes.byref(g)))
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=b.device) if nbytes else None
    if scratch is not None:
        g.workspace, g.workspace_bytes = scratch.data_ptr(), nbytes
    launch(name, index, _C.load().tnx_mx_gemm, g)
    del scratch
    return underived(name, out, *inputs)


def mx_matmul(a, b, out_dtype=None) -> torch.Tensor:
    """``a @ b`` of microscaled operands, ``a[m, k]`` quantised along k (``dim=-1``) and ``b[k, n]`` along k (``dim=-2``).

    Either may be a torch tensor, quantised on the way in.  32-bit sums, rounded once to ``out_dtype`` (default: ``a``'s dtype, bfloat16 where it
    has none).  No gradient passes: differentiating the result is an error where an operand asks for its own; ``mx_linear`` has them."""
    return _product("mx_matmul", a, b, out_dtype, _C.EPI_NONE)


def epilogue_of(activation: str) -> int:
    return _EPILOGUES.get(activation, _C.EPI_GLU_IDENTITY)


def mx_glu(x, w12, activation: str = "silu", out_dtype=None) -> torch.Tensor:
    """``act(x @ w12[:, 0::2]) * (x @ w12[:, 1::2])`` of microscaled operands: ``glu`` with the gate in the product's epilogue.  No gradient passes, as
    with ``mx_matmul``."""
    return _product("mx_glu", x, w12, out_dtype, epilogue_of(activation))


class _Linear(torch.autograd.Function):
    """What the native side has not taken; it keeps x and w themselves."""

    @staticmethod
    def forward(ctx, x, w):
        ctx.save_for_backward(x, w)
        return mx_matmul(x, w)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w = ctx.saved_tensors
        dx = dw = None
        if ctx.needs_input_grad[0]:
            dx = mx_matmul(dy, w.t(), out_dtype=x.dtype)
        if ctx.needs_input_grad[1]:
            dw = mx_matmul(x.t(), dy, out_dtype=w.dtype)
        return dx, dw


def mx_linear(x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    """``x[m, k] @ w[k, n]`` with all three products of a training step microscaled.

    Forward: x and w quantised along k.  Backward: ``dx = dy @ w^T`` with both quantised along n, ``dw = x^T @ dy`` with both
    quantised along m; the rounding of the operands counts as the identity.  For the backward pass x and w are kept quantised, as its products
    take them."""
    y = (native or find_native()).mx_linear(x, w)
    if y is not None:
        return y
    if x.dim() != 2 or w.dim() != 2 or x.shape[1] != w.shape[0]:
        raise ValueError(f"mx_linear expects x[m,k] and w[k,n], got {tuple(x.shape)} and {tuple(w.shape)}")
    if x.dtype != w.dtype:
        raise ValueError(f"mx_linear: x is {x.dtype}, w is {w.dtype}")
    return _Linear.apply(x, w)
