"""tnx_linear without a bias: what its bias_dtype holds does not count, whichever kernel runs."""
import ctypes

import pytest
import torch

import blocks_reference as ref
from tritonix_amd import _C

pytestmark = pytest.mark.gpu
CODES = {torch.float16: _C.F16, torch.bfloat16: _C.BF16, torch.float32: _C.F32}


@pytest.mark.parametrize("dtype", list(CODES))
@pytest.mark.parametrize("m,n,k,layout", [(3, 64, 96, "nt"), (2, 64, 4096, "nn"), (2, 9000, 64, "nn"), (70, 130, 96, "nn"), (40, 72, 33, "tn"), (600, 3000, 256, "nn")])
def test_the_type_of_no_bias(device, dtype, m, n, k, layout):
    x = ref.draw(device, k, m, dtype=dtype, seed=1).t() if layout == "tn" else ref.draw(device, m, k, dtype=dtype, seed=1)
    w = ref.draw(device, n, k, dtype=dtype, seed=2, scale=k ** -0.5).t() if layout == "nt" else ref.draw(device, k, n, dtype=dtype, seed=2, scale=k ** -0.5)
    lib, outs = _C.load(), []
    for kind in (CODES[dtype], -1, 77, (1 << 31) - 1, -(1 << 31)):
        y, z = torch.empty(m, n, dtype=dtype, device=device), torch.empty(m, n, dtype=dtype, device=device)
        a = _C.LinearArgs(x=x.data_ptr(), w=w.data_ptr(), y=y.data_ptr(), z=z.data_ptr(), m=m, n=n, k=k, stride_xm=x.stride(0), stride_xk=x.stride(1), stride_wk=w.stride(0),
                          stride_wn=w.stride(1), dtype=CODES[dtype], bias_dtype=kind, activation=_C.ACT_SILU, stream=torch.cuda.current_stream().cuda_stream)
        workspace = torch.zeros(lib.tnx_linear_workspace_bytes(ctypes.byref(a)) + 256, dtype=torch.uint8, device=device)
        scratch = torch.empty(lib.tnx_linear_scratch_bytes(ctypes.byref(a)) + 256, dtype=torch.uint8, device=device)
        a.workspace, a.workspace_bytes, a.scratch, a.scratch_bytes = workspace.data_ptr(), workspace.numel(), scratch.data_ptr(), scratch.numel()
        assert lib.tnx_linear(ctypes.byref(a)) == _C.OK
        torch.cuda.synchronize()
        outs.append((y, z))
    at = torch.arange(0, m, max(1, m // 20), device=device)
    ref.check("y", outs[0][0][at], ref.linear(x[at], w, None, "silu")["y"], dtype)
    for y, z in outs[1:]:
        assert torch.equal(y, outs[0][0]) and torch.equal(z, outs[0][1])
