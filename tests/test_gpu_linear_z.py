"""z = x w + bias as a linear layer keeps it for the backward pass, against the definition in 64 bits, from every kernel that writes it."""
import ctypes
import importlib

import pytest
import torch

import blocks_reference as ref
import tritonix
from tritonix_amd import _C

module = importlib.import_module("tritonix_amd.ops.linear")
pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
CODES = {torch.float16: _C.F16, torch.bfloat16: _C.BF16, torch.float32: _C.F32}

# m, n, k, layout of w (tn: row-major w, x contiguous along m)
SIZES = [(1, 1000, 704, "nt"), (4, 130, 1025, "nt"), (8, 4098, 640, "nt"), (8, 33, 4096, "nt"), (16, 129, 1025, "nt"), (2, 64, 4096, "nn"), (8, 1024, 4100, "nn"), (3, 9001, 1030, "nn"),
         (24, 4096, 4096, "nn"), (48, 512, 4096, "nt"), (64, 8192, 512, "nn"), (100, 1000, 600, "nt"), (256, 384, 5000, "nn"), (500, 3000, 256, "nt"), (1024, 1024, 1024, "nn"),
         (1500, 2000, 328, "nn"), (2048, 2048, 256, "nt"), (4096, 4096, 64, "nn"), (768, 5000, 192, "nn"), (5000, 700, 200, "nt"), (8192, 4096, 512, "nn"), (2500, 3001, 1000, "nt"),
         (4096, 2048, 2048, "nn"), (8192, 2112, 1024, "nt"), (3000, 2048, 1024, "nn"), (200, 264, 192, "nn"), (77, 90, 33, "tn"), (300, 520, 96, "tn"), (5, 40, 0, "nn")]


def operands(device, dtype, m, n, k, layout):
    x = ref.draw(device, k, m, dtype=dtype, seed=1).t() if layout == "tn" else ref.draw(device, m, k, dtype=dtype, seed=1)
    scale = max(k, 1) ** -0.5
    return x, ref.draw(device, n, k, dtype=dtype, seed=2, scale=scale).t() if layout == "nt" else ref.draw(device, k, n, dtype=dtype, seed=2, scale=scale)


def kernels(dtype):
    """{size: (route, tile, parts of k, scratch)} of the sizes above, from the host's choice."""
    lib, info, out = _C.load(), (ctypes.c_int32 * 5)(), {}
    for m, n, k, layout in SIZES:
        along_k, along_n = (1, k) if layout == "nt" else (n, 1)
        a = _C.LinearArgs(x=1 << 20, w=1 << 21, z=1 << 22, m=m, n=n, k=k, stride_xm=1 if layout == "tn" else k, stride_xk=m if layout == "tn" else 1, stride_wk=along_k,
                          stride_wn=along_n, dtype=CODES[dtype], bias_dtype=CODES[dtype], activation=_C.ACT_SILU)
        out[m, n, k, layout] = (lib.tnx_linear_route(ctypes.byref(a), info), tuple(info[:4]), info[4], lib.tnx_linear_scratch_bytes(ctypes.byref(a)))
    return out


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_sizes_reach_every_kind_of_kernel(dtype):
    made = kernels(dtype).values()
    assert {r for r, *_ in made} == {_C.LINEAR_ROUTE_FUSED, _C.LINEAR_ROUTE_APART, _C.LINEAR_ROUTE_STREAM, _C.LINEAR_ROUTE_STREAM_ROWS}
    fused = [v for v in made if v[0] == _C.LINEAR_ROUTE_FUSED]
    assert any(cut > 1 for _, _, cut, _ in fused) and any(cut <= 1 for _, _, cut, _ in fused)
    if dtype == torch.float32:
        # (on the binary32 instruction, and as heads and tails, for which the operands are cut into scratch)
        assert any(s == 0 for *_, s in fused) and any(s > 0 for *_, s in fused)
    else:
        assert len({t for _, t, _, _ in fused}) >= 8 and any(t[:2] == (256, 256) for _, t, _, _ in fused)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k,layout", SIZES)
def test_z(device, dtype, m, n, k, layout):
    x, w = operands(device, dtype, m, n, k, layout)
    bias, residual = ref.draw(device, n, dtype=dtype, seed=3), ref.draw(device, m, n, dtype=dtype, seed=4)
    # a sample of rows: the definition of all of them would take the CPU minutes
    at = torch.unique(torch.cat([torch.arange(0, m, max(1, m // 37)), torch.tensor([m - 1])])).to(device)
    for b, act, r in ((bias, "gelu", residual), (None, "silu", None), (bias.float(), None, residual)):
        y, z = module._run(x, w, b, r, module.ACTIVATIONS[act], True)
        ref.check(f"z {act}", z[at], ref.linear(x[at], w, b)["y"], dtype)
        ref.check(f"y {act}", y[at], ref.linear(x[at], w, b, act, None if r is None else r[at])["y"], dtype)
        # (writing z beside it changes nothing of y)
        assert torch.equal(y, tritonix.linear(x, w, b, act, r))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradients_through_a_large_tile(device, dtype):
    """dx and dbias of a layer on the largest tile, whose z the backward pass reads: a sample of rows, and of the sums over all rows a sample of columns."""
    m, n, k = 8192, 4096, 512
    x, w = operands(device, dtype, m, n, k, "nn")
    bias, dy = ref.draw(device, n, dtype=dtype, seed=3), ref.draw(device, m, n, dtype=dtype, seed=4)
    leaves = [t.requires_grad_(True) for t in (x, w, bias)]
    dx, dw, dbias = torch.autograd.grad(tritonix.linear(*leaves, "gelu"), leaves, dy)
    at = torch.arange(5, m, 409, device=device)
    ref.check("dx", dx[at], ref.linear(x[at], w, bias, "gelu", None, dy[at])["dx"], dtype)
    cols = torch.arange(3, n, 371, device=device)
    want = ref.linear(x, w[:, cols], bias[cols], "gelu", None, dy[:, cols])
    ref.check("dw", dw[:, cols], want["dw"], dtype)
    ref.check("dbias", dbias[cols], want["dbias"], dtype)
