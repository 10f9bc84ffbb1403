"""mx_glu's gate is glu's: of operands that are 4-bit floats already, whose products are exact, both give the same bits."""
import ctypes

import pytest
import torch

import tritonix
from tritonix_amd import _C

pytestmark = pytest.mark.gpu

LEVELS = torch.tensor([0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0])


def operands(m, n, k, seed):
    g = torch.Generator("cpu").manual_seed(seed)
    a, b = (LEVELS[torch.randint(0, len(LEVELS), s, generator=g)] for s in ((m, k), (k, n)))
    a[:, ::32], b[::32] = 4.0, 4.0                        # every block has the scale 1
    return a, b


def gated(a, b, activation, dtype):
    """The gated product on a tile of the wider types, in binary32; rounded once, it is the tile's result in 16 bits."""
    (m, k), n = a.shape, b.shape[1]
    a, b, z = a.bfloat16().contiguous(), b.bfloat16().contiguous(), torch.empty(m, n // 2, device=a.device)
    g = _C.GemmArgs()
    g.m, g.n, g.k = m, n, k
    g.stride_am, g.stride_ak, g.stride_bk, g.stride_bn, g.stride_cm, g.stride_cn = k, 1, n, 1, n // 2, 1
    g.in_dtype, g.out_dtype, g.epilogue = _C.BF16, _C.F32, {"silu": _C.EPI_GLU_SILU, "sigmoid": _C.EPI_GLU_SIGMOID, "none": _C.EPI_GLU_IDENTITY}[activation]
    g.block_m, g.block_n, g.block_k, g.num_warps, g.num_stages = 128, 128, 64, 8, 3
    g.split_k, g.group_m = 1, 8
    g.a, g.b, g.c, g.stream = a.data_ptr(), b.data_ptr(), z.data_ptr(), torch.cuda.current_stream().cuda_stream
    assert _C.load().tnx_gemm(ctypes.byref(g)) == _C.OK
    return z.to(dtype)


@pytest.mark.parametrize("size", [(4, 512, 64), (40, 700, 96), (300, 1030, 64), (1100, 2048, 64)], ids=str)
@pytest.mark.parametrize("activation", ["silu", "sigmoid", "none"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
def test_bits_of_glu(device, size, activation, dtype):
    m, n, k = size
    a, b = (t.to(dtype).to(device) for t in operands(m, n, k, m + n))
    want = gated(a, b, activation, dtype)
    z = (a.float() @ b.float())[:, 0::2]
    assert float(z.min()) < -88 and float(z.max()) > 88   # down to where the sigmoid is a subnormal number, and to zero
    for left in (a, tritonix.mx_quantize(a)):              # rows as floats, where the product takes them, and quantised
        got = tritonix.mx_glu(left, tritonix.mx_quantize(b, dim=0), activation, out_dtype=dtype)
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("tokens", [2, 200, 3000])
def test_bits_of_glu_by_expert(device, dtype, tokens):
    experts, d, f = 3, 64, 300
    x, _ = operands(tokens, 2, d, tokens)
    w = torch.stack([operands(1, 2 * f, d, e)[1] for e in range(experts)])
    x, w = x.to(dtype).to(device), w.to(dtype).to(device)
    chosen = torch.randint(0, experts, (tokens, 1), generator=torch.Generator("cpu").manual_seed(1)).to(device)
    r = tritonix.moe_plan(chosen, torch.ones(tokens, 1, device=device), experts)
    got = tritonix.moe_glu(x, tritonix.mx_quantize(w, dim=-2), r)
    assert got.dtype == dtype
    for e in range(experts):
        lo, hi = int(r.offsets[e]), int(r.offsets[e + 1])
        if lo < hi:
            assert torch.equal(got[lo:hi], gated(x[r.order[lo:hi].long()], w[e], "silu", dtype))
