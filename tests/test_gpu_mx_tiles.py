"""Every kernel of the microscaled products over more slabs of k than its ring of LDS buffers holds, with operands that differ from slab to slab.

A case names the kernel it is for, and the library is asked whether it takes it: a choice that moves on takes the test with it."""
import ctypes

import pytest
import torch

import tritonix
from tests import mx_reference as ref
from tritonix_amd import _C
from tritonix_amd.ops import mx

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, 0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], dtype=torch.float64)


def random_rows(device, rows, k, seed, exponent):
    """Codes and scales of rows as a checkpoint holds them, and what they stand for in 64 bits."""
    g = torch.Generator("cpu").manual_seed(seed)
    codes = torch.randint(0, 256, (rows, -(-k // 2)), generator=g, dtype=torch.uint8).to(device)
    scales = torch.randint(127 + exponent - 2, 127 + exponent + 2, (rows, -(-k // 32)), generator=g, dtype=torch.uint8).to(device)
    table = LEVELS.to(device)
    values = torch.stack([table[(codes & 15).long()], table[(codes >> 4).long()]], dim=2).flatten(1)[:, :k]
    return codes, scales, values * torch.exp2(scales.double() - 127).repeat_interleave(32, dim=1)[:, :k]


def rounding(want, dtype):
    bits, smallest = {torch.bfloat16: (8, 2.0 ** -133), torch.float16: (11, 2.0 ** -24), torch.float32: (24, 2.0 ** -149)}[dtype]
    return torch.exp2(torch.floor(torch.log2(want.abs().clamp(min=2.0 ** -200))) - bits).clamp(min=smallest / 2)


def product(a, b, k):
    """a @ b of values in 64 bits, and how far 32-bit sums of it may be (ref.product_bound)."""
    return a @ b, 2.0 ** -23 * (k / 32 + 8) * (a.abs() @ b.abs())


def gated(z, dz):
    """SiLU-gated columns and their bound (ref.gated)."""
    want, tol = ref.gated(z.cpu().numpy(), dz.cpu().numpy(), "silu")
    return torch.from_numpy(want).to(z.device), torch.from_numpy(tol).to(z.device)


def check(got, want, tol):
    tol = tol + rounding(want.abs() + tol, got.dtype)
    worst = float(((got.double() - want).abs() / tol).max())
    assert worst <= 1, worst                               # (a NaN is no such number)


def route_of(g):
    info = (ctypes.c_int32 * 4)()
    return _C.load().tnx_mx_gemm_route(ctypes.byref(g), info), tuple(info)


STREAM, TILES = 1, 2
# kernel (columns, rows, ring; parts of k): sizes of the product.  k: slabs past the ring by one and by many, odd counts and even ones, the last one part full
PLAIN = [((64, 64, 4, 1), (130, 1030, 1300)), ((64, 64, 4, 1), (70, 2050, 2600)), ((64, 64, 4, 5), (20, 2050, 5000)), ((64, 64, 4, 7), (63, 2050, 7000)), ((128, 128, 4, 8), (65, 3400, 28000)),
         ((128, 128, 4, 1), (1490, 2070, 1900)), ((128, 128, 4, 1), (200, 8200, 2600)), ((128, 128, 4, 1), (1020, 2050, 4100)),
         ((128, 128, 2, 1), (500, 8200, 800)), ((128, 128, 2, 1), (510, 8200, 1900)), ((256, 256, 2, 1), (1000, 8200, 800)), ((256, 256, 2, 1), (1100, 8100, 2600))]


@pytest.mark.parametrize("kernel,size", PLAIN, ids=str)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("epilogue", ["plain", "silu"])
def test_products(device, kernel, size, dtype, epilogue):
    m, n, k = size
    a_codes, a_scales, av = random_rows(device, m, k, m, -1)
    b_codes, b_scales, bv = random_rows(device, n, k, n + 1, -6)
    a, b = mx.MXTensor.from_codes(a_codes, a_scales, k), mx.MXTensor.from_codes(b_codes, b_scales, k, dim=-2)
    out = tritonix.mx_matmul(a, b, dtype) if epilogue == "plain" else tritonix.mx_glu(a, b, out_dtype=dtype)
    g = mx.gemm_args(a, b, out, _C.EPI_NONE if epilogue == "plain" else _C.EPI_GLU_SILU)
    room = _C.load().tnx_mx_gemm_workspace_bytes(ctypes.byref(g))
    if room:
        g.workspace, g.workspace_bytes = 256, room
    assert route_of(g) == (TILES, kernel)
    want, tol = product(av, bv.t().contiguous(), k)
    check(out, *((want, tol) if epilogue == "plain" else gated(want, tol)))


@pytest.mark.parametrize("size", [(5, 1000, 6000), (16, 300, 9000), (33, 200, 9000)], ids=str)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_streamed_weights(device, size, dtype):
    """The kernel without LDS buffers for the weights: more slabs than a turn of its waves."""
    m, n, k = size
    a_codes, a_scales, av = random_rows(device, m, k, m, -1)
    b_codes, b_scales, bv = random_rows(device, n, k, n + 1, -6)
    a, b = mx.MXTensor.from_codes(a_codes, a_scales, k), mx.MXTensor.from_codes(b_codes, b_scales, k, dim=-2)
    out = tritonix.mx_matmul(a, b, dtype)
    assert route_of(mx.gemm_args(a, b, out, _C.EPI_NONE))[0] == STREAM
    check(out, *product(av, bv.t().contiguous(), k))


# kernel: experts, rows of the product (two a token), width of the interleaved weights, k
EXPERTS = [((128, 32, 2, 1), (64, 140, 520, 800)), ((128, 32, 2, 1), (60, 300, 1030, 1900)), ((64, 64, 4, 1), (2, 40, 520, 1300)), ((64, 64, 4, 1), (3, 300, 262, 2600)),
           ((128, 128, 4, 1), (16, 1000, 1500, 1300)), ((128, 128, 4, 1), (16, 1000, 1500, 2600)), ((128, 128, 2, 1), (64, 4000, 520, 800)),
           ((128, 128, 2, 1), (64, 4000, 520, 1900)), ((256, 256, 2, 1), (8, 1100, 6100, 800)), ((256, 256, 2, 1), (3, 2000, 4100, 1900))]


@pytest.mark.parametrize("kernel,size", EXPERTS, ids=str)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_experts_products(device, kernel, size, dtype):
    """The gated product of gathered rows, and the plain one of rows as they lie: experts of uneven numbers of rows, one without any, and empty slots."""
    experts, rows, n, k = size
    tokens = rows // 2
    g = torch.Generator("cpu").manual_seed(rows)
    chosen = torch.randint(0, experts, (tokens, 2), generator=g)
    chosen[: tokens // 5, 0] = 0                           # a crowded expert,
    chosen[chosen == experts - 1] = -1                     # one without rows, and slots without an expert
    weights = [random_rows(device, n, k, 7 * e + 1, -6) for e in range(experts)]
    w = mx.MXTensor.from_codes(torch.stack([t[0] for t in weights]), torch.stack([t[1] for t in weights]), k, dim=-2)
    x_codes, x_scales, xv = random_rows(device, tokens, k, tokens, -1)
    h_codes, h_scales, hv = random_rows(device, 2 * tokens, k, tokens + 1, -1)
    r = tritonix.moe_plan(chosen.to(device), torch.ones(tokens, 2, device=device), experts)
    up = tritonix.moe_glu(mx.MXTensor.from_codes(x_codes, x_scales, k), w, r, out_dtype=dtype)
    h = mx.MXTensor.from_codes(h_codes, h_scales, k)
    down = torch.empty(2 * tokens, n, dtype=dtype, device=device)
    for args, gather in ((mx.gemm_args(mx.MXTensor.from_codes(x_codes, x_scales, k), w, up, _C.EPI_GLU_SILU), True), (mx.gemm_args(h, w, down, _C.EPI_NONE), False)):
        args.experts, args.offsets, args.top_k = experts, r.offsets.data_ptr(), 2
        if gather:
            args.order = r.order.data_ptr()
        assert route_of(args) == (TILES, kernel)
    args.stream = torch.cuda.current_stream().cuda_stream
    assert _C.load().tnx_mx_gemm(ctypes.byref(args)) == _C.OK
    offsets, order = r.offsets.tolist(), r.order.long()
    assert offsets[-1] < 2 * tokens and offsets[-1] == offsets[-2]
    assert bool((up[offsets[-1]:] == 0).all()) and bool((down[offsets[-1]:] == 0).all())
    for e in range(experts):
        lo, hi = offsets[e], offsets[e + 1]
        if lo < hi:
            wv = weights[e][2].t().contiguous()
            check(up[lo:hi], *gated(*product(xv[order[lo:hi] // 2], wv, k)))
            check(down[lo:hi], *product(hv[lo:hi], wv, k))
