"""What the microscaled and routing entry points refuse, and their host arithmetic: no GPU needed, nothing is launched."""
import ctypes
import os
import re

import pytest
import torch

import tritonix
from tritonix_amd import _C

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("struct,cls", [("tnx_mx_args", _C.MxArgs), ("tnx_mx_gemm_args", _C.MxGemmArgs), ("tnx_moe_args", _C.MoeArgs)])
def test_structs_are_the_headers(struct, cls):
    header = open(os.path.join(ROOT, "include", "tritonix_hip.h")).read()
    body = header[header.index(f"typedef struct {struct} {{") + len(f"typedef struct {struct} {{"):header.index(f"}} {struct};")]
    names = []
    for decl in re.sub(r"/\*.*?\*/", "", body, flags=re.S).split(";"):
        decl = re.sub(r"^(const\s+)?(void|int64_t|int32_t|float|size_t)\s*\*?", "", decl.strip())
        names += [n.strip(" *") for n in decl.split(",") if n.strip(" *")]
    assert names == [f[0] for f in cls._fields_]


def test_limits_are_the_headers():
    header = open(os.path.join(ROOT, "include", "tritonix_hip.h")).read()
    value = lambda name: int(re.search(rf"#define {name} (\d+)", header).group(1))      # noqa: E731
    assert (_C.MOE_MAX_EXPERTS, _C.MOE_MAX_TOP_K, _C.MOE_MAX_GROUPS) == tuple(
        value(n) for n in ("TNX_MOE_MAX_EXPERTS", "TNX_MOE_MAX_TOP_K", "TNX_MOE_MAX_GROUPS"))


def test_buffer_sizes():
    lib = _C.load()
    assert lib.tnx_mx_code_bytes(1, 1) == 128 and lib.tnx_mx_scale_bytes(1, 1) == 512
    assert lib.tnx_mx_code_bytes(33, 257) == 33 * 256 and lib.tnx_mx_scale_bytes(33, 257) == 2 * 512 and lib.tnx_mx_scale_bytes(32, 513) == 2 * 512
    assert lib.tnx_mx_code_bytes(80000, 131072) == 80000 * 65536
    assert lib.tnx_mx_code_bytes(0, 5) == lib.tnx_mx_scale_bytes(5, 0) == 0
    t = tritonix.MXTensor.empty(3, 33, 257, -2, "cpu")
    assert t.code_bytes == 3 * lib.tnx_mx_code_bytes(33, 257) and t.buffer.numel() - t.code_bytes == 3 * lib.tnx_mx_scale_bytes(33, 257)
    assert t.shape == (3, 257, 33) and t.t().shape == (3, 33, 257) and t.t().t().shape == t.shape
    # up to four tokens one workgroup does it all; then a count per block (four tokens, later 32) and expert, and a total per expert
    assert lib.tnx_moe_workspace_bytes(4, 8, 16) == 0 and lib.tnx_moe_workspace_bytes(5, 8, 16) == 16 * 2 * 4 + 16 * 4
    assert lib.tnx_moe_workspace_bytes(65536, 8, 128) == 2048 * 128 * 4 + 128 * 4


def mx(**kw):
    a = _C.MxArgs()
    for k, v in {**dict(data=256, codes=256, scales=256, batch=1, rows=4, k=64, stride_row=64, stride_k=1, dtype=_C.BF16), **kw}.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,status", [
    (dict(data=None), _C.E_INVALID), (dict(codes=264), _C.E_INVALID), (dict(scales=None), _C.E_INVALID), (dict(data=257), _C.E_INVALID),
    (dict(rows=-1), _C.E_INVALID), (dict(k=-1), _C.E_INVALID), (dict(batch=-1), _C.E_INVALID), (dict(dtype=_C.I8), _C.E_UNSUPPORTED),
    (dict(k=1 << 23), _C.E_UNSUPPORTED), (dict(batch=70000), _C.E_UNSUPPORTED), (dict(data=258, dtype=_C.F32), _C.E_INVALID),
    (dict(rows=0), _C.OK), (dict(k=0, data=None), _C.OK)])
def test_quantise_refuses(change, status):
    lib = _C.load()
    assert lib.tnx_mx_quantize(ctypes.byref(mx(**change))) == status
    assert lib.tnx_mx_dequantize(ctypes.byref(mx(**change))) == status
    assert lib.tnx_mx_quantize(None) == _C.E_INVALID


def gemm(**kw):
    g = _C.MxGemmArgs()
    for k, v in {**dict(a_codes=256, a_scales=256, b_codes=256, b_scales=256, out=256, m=4, n=8, k=64, a_rows=4, stride_out=8, out_dtype=_C.BF16), **kw}.items():
        setattr(g, k, v)
    return g


@pytest.mark.parametrize("change,status", [
    (dict(a_codes=None), _C.E_INVALID), (dict(b_scales=264), _C.E_INVALID), (dict(out=257), _C.E_INVALID), (dict(stride_out=7), _C.E_INVALID),
    (dict(m=-1), _C.E_INVALID), (dict(epilogue=4), _C.E_INVALID), (dict(out_dtype=_C.I32), _C.E_UNSUPPORTED), (dict(k=0), _C.E_UNSUPPORTED),
    (dict(n=7, epilogue=_C.EPI_GLU_SILU), _C.E_UNSUPPORTED), (dict(a_rows=3), _C.E_INVALID), (dict(experts=2), _C.E_INVALID),
    (dict(offsets=256), _C.E_INVALID), (dict(experts=2, offsets=256, order=256, a_rows=0, top_k=1), _C.E_INVALID),
    (dict(experts=2, offsets=256, order=256, top_k=0), _C.E_INVALID), (dict(experts=2000, offsets=256), _C.E_INVALID),
    (dict(k=1 << 23), _C.E_UNSUPPORTED), (dict(m=0), _C.OK), (dict(n=0), _C.OK), (dict(a_data=256), _C.E_INVALID),
    (dict(a_data=256, a_codes=None, a_scales=None, a_dtype=_C.BF16, m=17, a_rows=17), _C.E_UNSUPPORTED),
    (dict(a_data=257, a_codes=None, a_scales=None, a_dtype=_C.BF16, m=2, a_rows=2), _C.E_INVALID),
    (dict(a_data=256, a_codes=None, a_scales=None, a_dtype=_C.I8, m=2, a_rows=2), _C.E_UNSUPPORTED),
    (dict(a_data=256, a_codes=None, a_scales=None, a_dtype=_C.BF16, m=2, a_rows=2, k=31000), _C.E_UNSUPPORTED)])
def test_product_refuses(change, status):
    lib = _C.load()
    assert lib.tnx_mx_gemm(ctypes.byref(gemm(**change))) == status
    assert lib.tnx_mx_gemm(None) == _C.E_INVALID


def test_rows_that_the_product_takes_as_floats():
    lib = _C.load()
    assert [lib.tnx_mx_gemm_takes_rows(m, k) for m, k in (
        (1, 1), (1, 30720), (1, 30721), (2, 8192), (2, 8193), (16, 1024), (16, 1025), (17, 64), (0, 64), (1, 0))] == [1, 1, 0, 1, 0, 1, 0, 0, 0, 0]


def moe(**kw):
    a = _C.MoeArgs()
    base = dict(logits=256, weights=256, experts=256, offsets=256, order=256, rows=256, grad=256, grad_logits=256, tokens=4, stride_logits=8, num_experts=8,
                top_k=2, dtype=_C.BF16, num_groups=1, top_groups=1, group_top=1, scale=1.0)
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,status", [
    (dict(logits=None), _C.E_INVALID), (dict(weights=None), _C.E_INVALID), (dict(offsets=None), _C.E_INVALID), (dict(order=None), _C.E_INVALID),
    (dict(tokens=-1), _C.E_INVALID), (dict(top_k=0), _C.E_INVALID), (dict(top_k=9), _C.E_INVALID), (dict(num_experts=2000), _C.E_UNSUPPORTED),
    (dict(num_experts=64, top_k=40), _C.E_UNSUPPORTED), (dict(dtype=_C.I8), _C.E_UNSUPPORTED), (dict(scoring=2), _C.E_INVALID),
    (dict(num_groups=3), _C.E_INVALID), (dict(num_groups=4, top_groups=5), _C.E_INVALID), (dict(group_top=3), _C.E_INVALID),
    (dict(tokens=1 << 30), _C.E_UNSUPPORTED), (dict(tokens=5), _C.E_WORKSPACE), (dict(tokens=1000, workspace=256, workspace_bytes=16), _C.E_WORKSPACE),
    (dict(logits=257), _C.E_INVALID)])
def test_routing_refuses(change, status):
    lib = _C.load()
    assert lib.tnx_moe_route(ctypes.byref(moe(**change))) == status
    assert lib.tnx_moe_route(None) == lib.tnx_moe_plan(None) == lib.tnx_moe_route_backward(None) == _C.E_INVALID


@pytest.mark.parametrize("change,status", [(dict(grad=None), _C.E_INVALID), (dict(grad_logits=None), _C.E_INVALID), (dict(experts=None), _C.E_INVALID),
                                           (dict(scoring=-1), _C.E_INVALID), (dict(tokens=0, grad=None), _C.OK)])
def test_routing_gradient_refuses(change, status):
    assert _C.load().tnx_moe_route_backward(ctypes.byref(moe(**change))) == status


def test_import_and_combine_refuse():
    lib = _C.load()
    assert lib.tnx_mx_import(None, 256, 1, 4, 64, 256, 256, None) == _C.E_INVALID
    assert lib.tnx_mx_import(256, 256, 1, 4, 64, 257, 256, None) == _C.E_INVALID
    assert lib.tnx_mx_import(256, 256, -1, 4, 64, 256, 256, None) == _C.E_INVALID
    assert lib.tnx_mx_import(None, None, 1, 0, 64, None, None, None) == _C.OK
    assert lib.tnx_moe_combine(None, 256, 256, 256, 4, 2, 8, _C.BF16, _C.BF16, None) == _C.E_INVALID
    assert lib.tnx_moe_combine(256, 256, 256, 256, 4, 0, 8, _C.BF16, _C.BF16, None) == _C.E_INVALID
    assert lib.tnx_moe_combine(256, 256, 256, 256, 4, 2, 8, _C.I8, _C.BF16, None) == _C.E_UNSUPPORTED
    assert lib.tnx_moe_combine(256, 256, 256, 256, 4, 2, 8, _C.BF16, _C.I32, None) == _C.E_UNSUPPORTED
    assert lib.tnx_moe_combine(None, None, None, None, 0, 2, 8, _C.BF16, _C.BF16, None) == _C.OK


def test_python_refusals():
    x = torch.ones(4, 64)
    for call in (lambda: tritonix.mx_quantize(x), lambda: tritonix.mx_matmul(x, torch.ones(64, 8)), lambda: tritonix.moe_route(x, 2),
                 lambda: tritonix.moe_plan(torch.zeros(4, 2, dtype=torch.int32), torch.ones(4, 2), 8)):
        with pytest.raises(ValueError, match="HIP device"):
            call()
    w = tritonix.MXTensor.empty(None, 8, 64, -2, "cpu")
    e = tritonix.MXTensor.empty(3, 8, 64, -2, "cpu")
    z = torch.zeros(4, 2, dtype=torch.int32)
    r = tritonix.Routing(torch.ones(4, 2), z, torch.zeros(4, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), z, 3)
    for call in (lambda: tritonix.mx_quantize(x[0]), lambda: tritonix.mx_quantize(x, dim=2), lambda: tritonix.mx_quantize(x.int()),
                 lambda: tritonix.mx_matmul(x, w.t()), lambda: tritonix.mx_matmul(x[:, :32], w), lambda: tritonix.mx_matmul(x, e),
                 lambda: tritonix.mx_matmul(x, w, out_dtype=torch.int32), lambda: tritonix.mx_linear(x, torch.ones(32, 8)),
                 lambda: tritonix.mx_linear(x, torch.ones(64, 8).half()), lambda: tritonix.MXTensor.from_codes(x, x, 64),
                 lambda: tritonix.MXTensor.from_codes(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 3, dtype=torch.uint8), 64),
                 lambda: tritonix.moe_route(x, 65), lambda: tritonix.moe_route(x, 0), lambda: tritonix.moe_route(x[0], 1),
                 lambda: tritonix.moe_route(x, 33), lambda: tritonix.moe_route(x, 2, scoring="tanh"), lambda: tritonix.moe_route(x, 2, num_groups=5),
                 lambda: tritonix.moe_route(x, 2, num_groups=4, top_groups=5), lambda: tritonix.moe_route(x, 2, group_top=2),
                 lambda: tritonix.moe_route(x, 2, bias=torch.ones(63)), lambda: tritonix.moe_route(x, 2, bias=torch.ones(64).half()),
                 lambda: tritonix.moe_plan(z.float(), torch.ones(4, 2), 3), lambda: tritonix.moe_plan(z, torch.ones(4, 3), 3),
                 lambda: tritonix.moe_plan(z, torch.ones(4, 2), 0), lambda: tritonix.moe_glu(x, w, r), lambda: tritonix.moe_glu(x, e.t(), r),
                 lambda: tritonix.moe_glu(x[:3], e, r), lambda: tritonix.moe_down(x, e, r), lambda: tritonix.moe_ffn(x, e, e, r),
                 lambda: tritonix.moe_route_backward(torch.ones(4, 3), x, r)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("change,codes,scales,status", [
    (dict(batch=2), 256, 256, _C.E_INVALID), (dict(rows=-1), 256, 256, _C.E_INVALID), ({}, None, 256, _C.E_INVALID), ({}, 256, None, _C.E_INVALID),
    ({}, 264, 256, _C.E_INVALID), (dict(data=None), 256, 256, _C.E_INVALID), (dict(codes=None), 256, 256, _C.E_INVALID),
    (dict(scales=8), 256, 256, _C.E_INVALID), (dict(rows=1 << 23), 256, 256, _C.E_UNSUPPORTED), (dict(k=1 << 23), 256, 256, _C.E_UNSUPPORTED),
    (dict(dtype=_C.I8), 256, 256, _C.E_UNSUPPORTED), (dict(dtype=_C.I8, stride_row=3, stride_k=5), 256, 256, _C.E_UNSUPPORTED),
    (dict(rows=0), None, None, _C.OK), (dict(k=0, data=None), None, None, _C.OK)])
def test_both_quantisations_refuse(change, codes, scales, status):
    lib = _C.load()
    assert lib.tnx_mx_quantize_both(ctypes.byref(mx(**change)), codes, scales) == status
    assert lib.tnx_mx_quantize_both(None, 256, 256) == _C.E_INVALID


def test_workspace_of_a_product():
    lib = _C.load()

    def size(**kw):
        return lib.tnx_mx_gemm_workspace_bytes(ctypes.byref(gemm(**kw)))
    assert size() == size(m=8192, n=8192, k=8192) == size(m=0) == size(n=0) == size(m=100, n=4096, k=512) == 0
    bytes_of = size(m=100, n=4099, k=14336)                     # parts of 100 x 4100 floats
    assert bytes_of % 1640000 == 0 and 2 <= bytes_of // 1640000 <= 8
    assert size(m=100, n=4099, k=14336, experts=4, offsets=256) == 0 and size(m=1, n=4096, k=14336, a_data=256) == 0
    assert lib.tnx_mx_gemm_workspace_bytes(None) == 0
    assert lib.tnx_mx_gemm(ctypes.byref(gemm(workspace=264, workspace_bytes=1))) == _C.E_INVALID
