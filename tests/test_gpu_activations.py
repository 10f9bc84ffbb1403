"""Activations of linear layers at the ends of their range: infinities and huge numbers, and gelu where it is next to nothing."""
import ctypes

import pytest
import torch

import blocks_reference as ref
import tritonix
from tritonix_amd import _C
from tritonix_amd.ops.linear import ACTIVATIONS

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
CODES = {torch.float16: _C.F16, torch.bfloat16: _C.BF16, torch.float32: _C.F32}
INF = float("inf")

# m, n, k, how w (or x) lies, and the kernel that the sizes take: streamed columns, streamed rows, small and large tiles, the epilogue apart
PLACES = [(3, 64, 96, "nt", "stream"), (2, 64, 4096, "nn", "rows"), (2, 9000, 64, "nn", "rows"), (70, 130, 96, "nn", "fused"), (600, 3000, 256, "nn", "fused"),
          (4096, 512, 64, "nt", "fused"), (40, 72, 33, "tn", "apart")]
ROUTES = {"stream": _C.LINEAR_ROUTE_STREAM, "rows": _C.LINEAR_ROUTE_STREAM_ROWS, "fused": _C.LINEAR_ROUTE_FUSED, "apart": _C.LINEAR_ROUTE_APART}


def operands(device, dtype, m, n, k, layout):
    x = ref.draw(device, k, m, dtype=dtype, seed=1).t() if layout == "tn" else ref.draw(device, m, k, dtype=dtype, seed=1)
    w = ref.draw(device, n, k, dtype=dtype, seed=2, scale=k ** -0.5).t() if layout == "nt" else ref.draw(device, k, n, dtype=dtype, seed=2, scale=k ** -0.5)
    return x, w


def route_of(x, w, act):
    a = _C.LinearArgs(x=x.data_ptr(), w=w.data_ptr(), bias=w.data_ptr(), m=x.shape[0], n=w.shape[1], k=x.shape[1], stride_xm=x.stride(0), stride_xk=x.stride(1),
                      stride_wk=w.stride(0), stride_wn=w.stride(1), dtype=CODES[x.dtype], bias_dtype=_C.F32, activation=ACTIVATIONS[act])
    return _C.load().tnx_linear_route(ctypes.byref(a), None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("m,n,k,layout,place", PLACES)
def test_infinities_have_their_limits(device, dtype, act, m, n, k, layout, place):
    """z of +inf and -inf, and numbers next to the largest: the activation's limits, +inf (or z) and zero, and the slope's, one and zero; the columns beside them are
    what they were, a NaN stays one."""
    if place == "rows" and (dtype == torch.float32) != (n == 9000):
        pytest.skip("other sizes stream a row-major weight of this type")
    x, w = operands(device, dtype, m, n, k, layout)
    assert route_of(x, w, act) == ROUTES[place]
    bias = ref.draw(device, n, dtype=torch.float32, seed=3)
    clean = tritonix.linear(x, w, bias, act)
    huge = {torch.float16: 6e4, torch.bfloat16: 1e38, torch.float32: 1e38}[dtype]
    bias[0], bias[5], bias[n - 1], bias[n - 2], bias[7] = INF, -INF, -huge, huge, float("nan")
    leaves = [t.detach().requires_grad_(True) for t in (x, w, bias)]
    y = tritonix.linear(leaves[0], leaves[1], leaves[2], act)
    dy = ref.draw(device, m, n, dtype=dtype, seed=4)
    (dbias,) = torch.autograd.grad(y, leaves[2:], dy)
    y = y.detach()
    assert torch.isposinf(y[:, 0]).all() and (y[:, 5] == 0).all() and (y[:, n - 1] == 0).all() and y[:, 7].isnan().all()
    assert (y[:, n - 2].double() - huge).abs().max() <= 2 * ref.unit(dtype) * huge + 100        # (z is huge and a product of order one)
    others = [c for c in range(n) if c not in (0, 5, 7, n - 2, n - 1)]
    assert torch.equal(y[:, others], clean[:, others]) and torch.equal(tritonix.linear(x, w, bias, act)[:, others], clean[:, others])
    # the bias' gradient is the sum of dy times the slope: of dy itself, or nothing
    total, magnitude = dy.double().sum(dim=0), dy.double().abs().sum(dim=0)
    for c in (0, n - 2):
        assert (dbias[c].double() - total[c]).abs() <= (m + 2) * ref.E * magnitude[c]
    assert dbias[5] == 0 and dbias[n - 1] == 0 and dbias[7].isnan()


def gelu_exactly(z):
    return 0.5 * z * torch.special.erfc(-z * 0.5 ** 0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("place", ["stream", "fused", "apart"])
def test_gelu_below_zero_is_relatively_exact(device, dtype, place):
    """From -12 to next to 0, where it falls to 1e-32, gelu and its slope are off by what 32-bit arithmetic costs, relative to themselves.

    With e^-(z^2 / 2) from one exponential of a rounded argument: z^2 times half a step, times log2 e (rounded, and the constant's own 0.1 steps), is 1.11 z^2 / 2 steps of the result; the
    exponential's and the reciprocal's last step, a polynomial of eight terms whose magnitudes add up to 1.65 (two half steps each) and four products come to 12 steps more, the polynomial's own error
    to 1.6: in all (14 + 1.2 z^2 / 2) E.  The slope is the difference of two such terms, of 1.3 times its own size together from -3 on down."""
    m, n, k = {"stream": (8 if dtype == torch.float32 else 16, 16, 16), "fused": (2048, 64, 64), "apart": (2048, 16, 33)}[place]
    z = torch.linspace(-12, -0.01, m).to(dtype).double()
    x, w = torch.zeros(m, k, dtype=dtype, device=device), torch.zeros(k, n, dtype=dtype, device=device)
    x[:, 0], w[0, 0] = z.to(dtype).to(device), 1.0
    if place == "apart":
        x = x.t().contiguous().t()
    elif place == "stream":
        w = w.t().contiguous().t()
    assert route_of(x, w, "gelu") == ROUTES[place]
    x.requires_grad_(True)
    y = tritonix.linear(x, w, None, "gelu")
    dy = torch.zeros(m, n, dtype=dtype, device=device)
    dy[:, 0] = 1.0
    (dx,) = torch.autograd.grad(y, x, dy)
    steps = (14 + 0.6 * z * z) * ref.E
    want = gelu_exactly(z)
    ref.check("gelu", y[:, 0], (want, steps * want.abs() + ref.rounding(want, dtype)))
    slope = 0.5 * torch.special.erfc(-z * 0.5 ** 0.5) + z * torch.exp(-0.5 * z * z) * (2 * torch.pi) ** -0.5
    # (dz is rounded for the product dx = dz w^T, and dx once more; above -3 the terms cancel: their magnitudes)
    terms = 0.5 * torch.special.erfc(-z * 0.5 ** 0.5) + z.abs() * torch.exp(-0.5 * z * z) * (2 * torch.pi) ** -0.5
    ref.check("slope", dx[:, 0], (slope, steps * torch.where(z <= -3, 1.3 * slope.abs(), terms) + 2 * ref.rounding(slope, dtype) + (k + 2) * ref.E * slope.abs()))
