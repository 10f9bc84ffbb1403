"""Linear layers, layer normalisation and grouped products without a GPU: what is refused, and the host's choices."""
import ctypes
import itertools

import pytest
import torch

import tritonix
from tritonix_amd import _C

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def t(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("call,text", [
    (lambda: tritonix.linear(t(4, 8), t(9, 6)), "expects"),
    (lambda: tritonix.linear(t(4, 8), t(8)), "expects"),
    (lambda: tritonix.linear(t(4, 8), t(2, 8, 6)), "expects"),
    (lambda: tritonix.linear(t(), t(8, 6)), "expects"),
    (lambda: tritonix.linear(t(4, 8), t(8, 6, dtype=F16)), "float16"),
    (lambda: tritonix.linear(t(4, 8, dtype=torch.int8), t(8, 6, dtype=torch.int8)), "int8"),
    (lambda: tritonix.linear(t(4, 8, dtype=torch.float64), t(8, 6, dtype=torch.float64)), "float64"),
    (lambda: tritonix.linear(t(4, 8), t(8, 6), t(8)), "bias"),
    (lambda: tritonix.linear(t(4, 8), t(8, 6), t(1, 6)), "bias"),
    (lambda: tritonix.linear(t(4, 8), t(8, 6), t(6, dtype=F16)), "bias"),
    (lambda: tritonix.linear(t(4, 8), t(8, 6), residual=t(6)), "residual"),
    (lambda: tritonix.linear(t(4, 8), t(8, 6), residual=t(1, 6)), "residual"),
    (lambda: tritonix.linear(t(4, 8), t(8, 6), residual=t(4, 6, dtype=F32)), "residual"),
    (lambda: tritonix.linear(t(4, 8), t(8, 6), activation="tanh"), "activation"),
    (lambda: tritonix.linear(t(4, 8), t(8, 6), activation="none"), "activation"),
    (lambda: tritonix.linear(t(4, 8), t(8, 6)), "HIP device"),
    (lambda: tritonix.layer_norm(t(4, 8), t(7)), "weight"),
    (lambda: tritonix.layer_norm(t(4, 8), t(8, dtype=F16)), "weight"),
    (lambda: tritonix.layer_norm(t(4, 8), t(8), t(4, 8)), "bias"),
    (lambda: tritonix.layer_norm(t(4, 8, dtype=torch.int32)), "int32"),
    (lambda: tritonix.layer_norm(t(4, 8), eps=-1e-5), "eps"),
    (lambda: tritonix.layer_norm(t(4, 8), eps=float("nan")), "eps"),
    (lambda: tritonix.layer_norm(t()), "scalar"),
    (lambda: tritonix.layer_norm(t(4, 8)), "HIP device"),
    (lambda: tritonix.grouped_matmul(t(4, 8), t(2, 9, 6), t(3, dtype=torch.int32)), "expects"),
    (lambda: tritonix.grouped_matmul(t(4, 8), t(8, 6), t(3, dtype=torch.int32)), "expects"),
    (lambda: tritonix.grouped_matmul(t(1, 4, 8), t(2, 8, 6), t(3, dtype=torch.int32)), "expects"),
    (lambda: tritonix.grouped_matmul(t(4, 8), t(2, 8, 6), t(2, dtype=torch.int32)), "offsets"),
    (lambda: tritonix.grouped_matmul(t(4, 8), t(2, 8, 6), t(3, dtype=F32)), "offsets"),
    (lambda: tritonix.grouped_matmul(t(4, 8), t(2, 8, 6, dtype=F16), t(3, dtype=torch.int32)), "float16"),
    (lambda: tritonix.grouped_matmul(t(4, 8), t(0, 8, 6), t(1, dtype=torch.int32)), "groups"),
    (lambda: tritonix.grouped_matmul(t(1, 1), t(4097, 1, 1), t(4098, dtype=torch.int32)), "groups"),
    (lambda: tritonix.grouped_matmul(t(4, 8), t(2, 8, 6), t(3, dtype=torch.int32)), "HIP device"),
])
def test_refusals(call, text):
    with pytest.raises(ValueError, match=text):
        call()


def linear_args(m, n, k, dtype=_C.BF16, layout="nn", epilogue=True):
    a = _C.LinearArgs()
    a.x, a.w = 1 << 20, 1 << 21                              # (only their alignment counts)
    a.m, a.n, a.k, a.dtype, a.bias_dtype = m, n, k, dtype, dtype
    a.stride_xm, a.stride_xk = k, 1
    a.stride_wk, a.stride_wn = (n, 1) if layout == "nn" else (1, k)
    a.activation = _C.ACT_SILU if epilogue else _C.ACT_NONE
    return a


@pytest.mark.parametrize("dtype", [_C.BF16, _C.F16, _C.F32])
@pytest.mark.parametrize("layout", ["nn", "nt"])
def test_every_choice_of_tile_has_the_epilogue(dtype, layout):
    lib = _C.load()
    tiles = set()
    for m, n, k in itertools.product((1, 7, 16, 33, 64, 65, 100, 200, 300, 513, 1000, 1600, 2500, 4096, 8192), (16, 64, 96, 130, 500, 768, 1111, 2048, 3000, 4096, 14336),
                                     (8, 64, 72, 200, 512, 1000, 2048, 4096, 5000, 14336)):
        info = (ctypes.c_int32 * 5)()
        route = lib.tnx_linear_route(ctypes.byref(linear_args(m, n, k, dtype, layout)), info)
        if route == (_C.LINEAR_ROUTE_STREAM if layout == "nt" else _C.LINEAR_ROUTE_STREAM_ROWS) and m <= (16 if layout == "nt" else 8):
            continue
        assert route == _C.LINEAR_ROUTE_FUSED, (m, n, k, list(info))
        tiles.add(tuple(info[:4]))
    assert len(tiles) >= (5 if dtype == _C.F32 else 12), tiles


def test_routes_of_a_linear_layer():
    lib = _C.load()
    route = lambda a: lib.tnx_linear_route(ctypes.byref(a), None)  # noqa: E731
    assert route(linear_args(100, 200, 300, epilogue=False)) == _C.LINEAR_ROUTE_PRODUCT
    a = linear_args(100, 200, 304)
    a.stride_xm, a.stride_xk = 1, 100                         # contiguous along m
    assert route(a) == _C.LINEAR_ROUTE_APART and lib.tnx_linear_scratch_bytes(ctypes.byref(a)) >= 100 * 200 * 4
    assert route(linear_args(100, 200, 0)) == _C.LINEAR_ROUTE_APART
    for m, n, k in ((1, 1, 1), (1, 100000, 4096), (4, 200, 8192), (8, 4096, 4096), (16, 2000, 2816), (4, 1000, 701)):
        few = linear_args(m, n, k, layout="nt")
        assert route(few) == _C.LINEAR_ROUTE_STREAM and lib.tnx_linear_workspace_bytes(ctypes.byref(few)) == 0
    for m, n, k in ((17, 200, 304), (16, 512, 8192), (16, 512, 2824), (8, 200, 8192), (4, 14336, 4096), (1, 4096, 14336), (4, 4096, 1001)):
        assert route(linear_args(m, n, k, layout="nt")) == _C.LINEAR_ROUTE_FUSED, (m, n, k)
    assert route(linear_args(4, 200, 304, _C.F32, "nt")) == route(linear_args(8, 4096, 4096, _C.F32, "nt")) == _C.LINEAR_ROUTE_STREAM
    assert route(linear_args(4, 20000, 304, _C.F32)) == _C.LINEAR_ROUTE_STREAM_ROWS
    for other in (linear_args(9, 200, 304, _C.F32, "nt"), linear_args(8, 200, 4616, _C.F32, "nt"), linear_args(5, 20000, 304, _C.F32), linear_args(4, 20000, 4104, _C.F32), linear_args(4, 8192, 304, _C.F32),
                  linear_args(16, 200, 304, _C.F32, "nt"), linear_args(4, 200, 8200, _C.F32, "nt")):
        assert route(other) == _C.LINEAR_ROUTE_FUSED
    for m, n, k in ((1, 8, 4096), (8, 1024, 4100), (4, 200, 8192), (4, 8, 4096)):
        few = linear_args(m, n, k)
        assert route(few) == _C.LINEAR_ROUTE_STREAM_ROWS
        need = lib.tnx_linear_workspace_bytes(ctypes.byref(few))
        assert need >= _C.WS_COUNTER_BYTES + 8 * 4 * m * n, (m, n, k, need)
        few.y = 1 << 22                                       # refused before any launch: without its workspace, with one too short, with one off 16 bytes
        assert lib.tnx_linear(ctypes.byref(few)) == _C.E_WORKSPACE
        few.workspace, few.workspace_bytes = 1 << 23, need - 1
        assert lib.tnx_linear(ctypes.byref(few)) == _C.E_WORKSPACE
        few.workspace, few.workspace_bytes = (1 << 23) + 8, need
        assert lib.tnx_linear(ctypes.byref(few)) == _C.E_WORKSPACE
    for m, n, k in ((9, 200, 4096), (1, 1025, 4096), (1, 200, 4095), (1, 7, 4096)):
        assert route(linear_args(m, n, k)) == _C.LINEAR_ROUTE_FUSED, (m, n, k)
    assert route(linear_args(0, 200, 300)) == 0
    bad = linear_args(100, 200, 300)
    bad.activation = 5
    assert route(bad) == 0 and lib.tnx_linear(ctypes.byref(bad)) == _C.E_INVALID
    other = linear_args(100, 200, 300, dtype=_C.I8)
    assert lib.tnx_linear(ctypes.byref(other)) == _C.E_UNSUPPORTED
    bias = linear_args(100, 200, 300)
    bias.bias, bias.bias_dtype, bias.y = 1 << 20, _C.F16, 1 << 20
    assert lib.tnx_linear(ctypes.byref(bias)) == _C.E_UNSUPPORTED
    cut = linear_args(16, 512, 8192)
    cut.y = 1 << 20
    assert lib.tnx_linear_workspace_bytes(ctypes.byref(cut)) > _C.WS_COUNTER_BYTES and lib.tnx_linear(ctypes.byref(cut)) == _C.E_WORKSPACE
    assert lib.tnx_linear(None) == _C.E_INVALID


def test_entry_points_refuse():
    lib = _C.load()
    a = _C.NormArgs(rows=4, n=8, dtype=_C.I8)
    assert lib.tnx_layer_norm(ctypes.byref(a)) == _C.E_UNSUPPORTED
    a = _C.NormArgs(x=4096, y=4096, rows=4, n=8, dtype=_C.BF16, weight=4096, weight_dtype=_C.F16)
    assert lib.tnx_layer_norm(ctypes.byref(a)) == _C.E_UNSUPPORTED
    a = _C.NormArgs(x=4096, y=4096, rows=4, n=8, dtype=_C.BF16, mean=4096)          # one of the statistics without the other
    assert lib.tnx_layer_norm(ctypes.byref(a)) == _C.E_INVALID
    a = _C.NormArgs(rows=4, n=8, dtype=_C.BF16, eps=-1.0)
    assert lib.tnx_layer_norm(ctypes.byref(a)) == _C.E_INVALID
    a = _C.NormArgs(x=4096, dy=4096, mean=4096, rstd=4096, dx=4096, dweight=4096, rows=400, n=8, dtype=_C.BF16, weight_dtype=_C.BF16)
    assert lib.tnx_layer_norm_workspace_bytes(ctypes.byref(a)) > 0 and lib.tnx_layer_norm_backward(ctypes.byref(a)) == _C.E_WORKSPACE
    g = _C.LinearGradientArgs(dy=4096, dbias=4096, m=400, n=8, dtype=_C.BF16, bias_dtype=_C.BF16)
    assert lib.tnx_linear_gradient_bytes(ctypes.byref(g)) > 0 and lib.tnx_linear_gradient(ctypes.byref(g)) == _C.E_WORKSPACE
    g = _C.LinearGradientArgs(dy=4096, dz=4096, m=400, n=8, dtype=_C.BF16, activation=_C.ACT_SILU)
    assert lib.tnx_linear_gradient(ctypes.byref(g)) == _C.E_INVALID                 # the derivative needs z


def grouped_args(**more):
    return _C.GroupedArgs(**{**dict(a=4096, b=4096, c=4096, offsets=4096, rows=100, n=64, k=64, stride_ar=64, stride_ak=1, stride_group=4096, stride_bk=64,
                                    stride_bn=1, groups=3, dtype=_C.BF16), **more})


def test_grouped_entry_point_refuses():
    lib = _C.load()
    for status, more in ((_C.E_INVALID, dict(form=2)), (_C.E_INVALID, dict(groups=0)), (_C.E_INVALID, dict(rows=-1)), (_C.E_INVALID, dict(offsets=None)),
                         (_C.E_UNSUPPORTED, dict(dtype=_C.I8)), (_C.E_UNSUPPORTED, dict(groups=5000)), (_C.E_UNSUPPORTED, dict(stride_ak=2)),
                         (_C.E_UNSUPPORTED, dict(stride_ar=63)), (_C.E_UNSUPPORTED, dict(stride_bn=2)), (_C.E_UNSUPPORTED, dict(block_m=96, block_n=96)),
                         (_C.E_UNSUPPORTED, dict(form=_C.GROUPED_WEIGHT_GRADIENT, n=3, stride_bk=3)), (_C.E_UNSUPPORTED, dict(n=3, k=65, stride_ar=65, stride_bk=3))):
        assert lib.tnx_grouped(ctypes.byref(grouped_args(**more))) == status, more
    info = (ctypes.c_int32 * 5)()
    assert lib.tnx_grouped_route(ctypes.byref(grouped_args()), info) == 1 and info[3] == 0
    few = dict(rows=12, stride_bk=1, stride_bn=64)
    assert lib.tnx_grouped_route(ctypes.byref(grouped_args(**few)), info) == 2 and list(info) == [0] * 5
    assert lib.tnx_grouped_workspace_bytes(ctypes.byref(grouped_args(**{**few, "k": 4096, "stride_ar": 4096, "stride_bn": 4096}))) == 0
    long = dict(rows=8, k=4096, stride_ar=4096)
    assert lib.tnx_grouped_route(ctypes.byref(grouped_args(**long)), info) == 2 and list(info) == [0, 0, 0, 0, 8]
    need = lib.tnx_grouped_workspace_bytes(ctypes.byref(grouped_args(**long)))
    assert need == 8 * 8 * 64 * 4
    for workspace, length in ((4096, need - 1), (4104, need)):
        assert lib.tnx_grouped(ctypes.byref(grouped_args(**long, workspace=workspace, workspace_bytes=length))) == _C.E_WORKSPACE
    for more in (dict(rows=9), dict(k=1023, stride_ar=1023), dict(n=4096 + 64, stride_bk=4096 + 64)):
        assert lib.tnx_grouped_route(ctypes.byref(grouped_args(**{**long, **more})), info) == 1, more
    assert lib.tnx_grouped_route(ctypes.byref(grouped_args(**few, dtype=_C.F32)), info) == 2
    for more in (dict(rows=13), dict(block_m=64, block_n=64), dict(form=_C.GROUPED_WEIGHT_GRADIENT, stride_bk=64, stride_bn=1)):
        assert lib.tnx_grouped_route(ctypes.byref(grouped_args(**{**few, **more})), info) == 1, more
    for more in (dict(stride_ar=63), dict(stride_bn=63), dict(stride_ak=2)):
        assert lib.tnx_grouped(ctypes.byref(grouped_args(**{**few, **more}))) == _C.E_UNSUPPORTED, more
    for more in (dict(k=63, stride_ar=63), dict(n=63, stride_bk=63), dict(a=4098), dict(b=4100), dict(stride_group=4097)):
        assert lib.tnx_grouped_route(ctypes.byref(grouped_args(**more)), info) == 1 and info[3] == 1, more


def test_accumulators_stay_in_registers():
    """No kernel of a linear layer or a grouped product keeps its sums in memory: what the compiler reported of them."""
    import json
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "build", "kernel_resources.json")
    if not os.path.exists(path):
        pytest.skip("no build report (the library was built elsewhere)")
    with open(path) as f:
        report = json.load(f)
    scratch = {k: v["scratch"] for k, v in report.items() if k.endswith((" linear", " grouped"))}
    # (256x256 tiles fill every register with sums and fragments: what little they spill is worked out before their loop)
    assert {k: v for k, v in scratch.items() if v > (80 if "256x256" in k and not k.endswith("64 w8 s2 bt linear") else 0)} == {}
