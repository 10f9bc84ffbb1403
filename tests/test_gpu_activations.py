"""Activations of linear layers at the ends of their range: infinities and huge numbers."""
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
