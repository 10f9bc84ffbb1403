"""Grouped products of more tiles than a grid's threads, counted in 32 bits, hold: refused, or given a tile that they hold."""
import ctypes

import pytest

from tritonix_amd import _C

THREADS = 1 << 32


def args(rows, groups, k, n, dtype=_C.BF16, form=_C.GROUPED_ROWS, **more):
    b = dict(stride_group=k * n, stride_bk=n, stride_bn=1)
    return _C.GroupedArgs(**{**dict(a=4096, b=4096, c=4096, offsets=4096, rows=rows, n=n, k=k, stride_ar=k, stride_ak=1, groups=groups, dtype=dtype, form=form), **b, **more})


def route(a):
    info = (ctypes.c_int32 * 5)()
    return _C.load().tnx_grouped_route(ctypes.byref(a), info), list(info)


def threads(a, info):
    bm, bn, waves, _, parts = info
    down = a.groups * -(-a.k // bm) if a.form == _C.GROUPED_WEIGHT_GRADIENT else a.rows // bm + min(a.groups + 2, a.rows)
    return down * -(-a.n // bn) * max(parts, 1) * waves * 64


TOO_MANY = [args(4096, 4096, 64, 1 << 20), args(1 << 20, 4096, 8, 1 << 22), args(100, 4096, 8, 1 << 20, form=_C.GROUPED_WEIGHT_GRADIENT),
            args(1 << 22, 4, 64, 8192, block_m=32, block_n=64), args(4096, 4096, 64, 1 << 19, _C.F32), args(1 << 29, 4096, 1 << 29, 1 << 29),
            args(1 << 29, 4096, 1 << 29, 1 << 29, block_m=64, block_n=64, parts=(1 << 31) - 1), args(5, 4096, 1 << 29, 1 << 29, form=_C.GROUPED_WEIGHT_GRADIENT)]


@pytest.mark.parametrize("case", range(len(TOO_MANY)))
def test_too_many_are_refused(case):
    a = TOO_MANY[case]
    lib = _C.load()
    assert route(a)[0] == 0
    assert lib.tnx_grouped(ctypes.byref(a)) == _C.E_UNSUPPORTED


def test_a_choice_is_one_that_the_grid_holds():
    sizes = [(4096, 4096, 64, 1 << n) for n in range(6, 19)] + [(1 << m, 64, 64, 16384) for m in range(10, 23)] + [(1 << 20, 1024, 8, 1 << n) for n in range(10, 18)]
    for rows, groups, k, n in sizes:
        for form in (_C.GROUPED_ROWS, _C.GROUPED_WEIGHT_GRADIENT):
            a = args(rows, groups, k, n, form=form)
            found, info = route(a)
            assert found == 1 and threads(a, info) < THREADS, (rows, groups, k, n, form, info)
