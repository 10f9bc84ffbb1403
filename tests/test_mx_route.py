"""Which kernel a microscaled product takes, asked of the library: host arithmetic, no GPU needed."""
import ctypes

import pytest

from tests.test_gpu_mx_tiles import EXPERTS, PLAIN, STREAM, TILES, route_of
from tests.test_mx_host import gemm
from tritonix_amd import _C


def sizes(m, n, k, **kw):
    g = gemm(m=m, n=n, k=k, a_rows=m, stride_out=n, **kw)
    room = _C.load().tnx_mx_gemm_workspace_bytes(ctypes.byref(g))
    if room:
        g.workspace, g.workspace_bytes = 256, room
    return g


def test_tested_sizes_take_the_kernels_they_are_for():
    for kernel, (m, n, k) in PLAIN:
        for epilogue in (_C.EPI_NONE, _C.EPI_GLU_SILU):
            assert route_of(sizes(m, n, k, epilogue=epilogue)) == (TILES, kernel)
    for kernel, (experts, m, n, k) in EXPERTS:
        assert route_of(sizes(m, n, k, experts=experts, offsets=256)) == (TILES, kernel)


def test_every_kernel_has_its_cases():
    """Of the kernels that the choice can take, each with more slabs of k than its ring has buffers, and those that cut k."""
    for cases, kernels in ((PLAIN, {(64, 64, 4), (128, 128, 4), (128, 128, 2), (256, 256, 2)}), (EXPERTS, {(128, 32, 2), (64, 64, 4), (128, 128, 4), (128, 128, 2), (256, 256, 2)})):
        assert {kernel[:3] for kernel, size in cases if kernel[3] == 1 and -(-size[-1] // 256) > kernel[2]} == kernels
    assert {kernel[:3] for kernel, _ in PLAIN if kernel[3] > 1} == {(64, 64, 4), (128, 128, 4)}
    seen = set()
    for k in (256, 1300, 4100, 14336, 28672):
        for m in (1, 8, 17, 40, 65, 130, 300, 1025, 4099, 8192):
            for n in (16, 70, 520, 2050, 4096, 14336):
                seen.add((False, route_of(sizes(m, n, k))[1][:3]))
                for experts in (4, 16, 64, 128):
                    seen.add((True, route_of(sizes(m, n, k, experts=experts, offsets=256))[1][:3]))
    assert seen <= {(False, kernel[:3]) for kernel, _ in PLAIN} | {(True, kernel[:3]) for kernel, _ in EXPERTS} | {(False, (16, 16, 0))}


@pytest.mark.parametrize("rows,experts", [(1, 0), (16, 0), (1, 8), (4, 64)])
def test_rows_as_floats_are_streamed(rows, experts):
    kw = dict(experts=experts, offsets=256, order=256, top_k=2) if experts else {}
    g = gemm(a_codes=None, a_scales=None, a_data=256, a_dtype=_C.BF16, m=rows * (2 if experts else 1), a_rows=rows, n=4096, k=1024, stride_out=4096, stride_a=1024, **kw)
    assert route_of(g) == (STREAM, (16, 16, 0, 1))


def test_what_is_refused_or_empty_has_no_kernel():
    for change in (dict(a_codes=None), dict(b_scales=264), dict(k=0), dict(n=7, epilogue=_C.EPI_GLU_SILU), dict(out_dtype=_C.I32), dict(m=0, a_rows=0), dict(n=0)):
        assert route_of(gemm(**change))[0] == 0
    lib = _C.load()
    assert lib.tnx_mx_gemm_route(None, None) == 0 and lib.tnx_mx_gemm_route(ctypes.byref(gemm()), None) in (STREAM, TILES)


def test_scratch_decides_whether_k_is_cut():
    cut, whole = sizes(100, 4096, 14336), gemm(m=100, n=4096, k=14336, a_rows=100, stride_out=4096)
    assert route_of(cut)[1][3] > 1 and route_of(whole)[1][3] == 1
