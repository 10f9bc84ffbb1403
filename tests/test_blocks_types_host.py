"""Types that the entry points of linear layers and normalisation are given beside pointers: those of what is not given do not count, those of what is asked for do."""
import ctypes

import pytest

from tritonix_amd import _C


@pytest.mark.parametrize("name", ["weight", "bias"])
@pytest.mark.parametrize("dtype", [_C.F16, _C.I8, -1, 77])
def test_a_parameters_gradient_has_a_type(name, dtype):
    """dweight without weight and dbias without bias: of the rows' type or float32, or refused ahead of any launch."""
    lib = _C.load()
    a = _C.NormArgs(x=4096, dy=4096, mean=4096, rstd=4096, rows=400, n=8, dtype=_C.BF16, eps=1e-5, **{"d" + name: 4096, name + "_dtype": dtype})
    assert lib.tnx_layer_norm_backward(ctypes.byref(a)) == _C.E_UNSUPPORTED
    assert lib.tnx_layer_norm_workspace_bytes(ctypes.byref(a)) == 0
    for good in (_C.BF16, _C.F32):
        setattr(a, name + "_dtype", good)
        assert lib.tnx_layer_norm_workspace_bytes(ctypes.byref(a)) > 0
        assert lib.tnx_layer_norm_backward(ctypes.byref(a)) == _C.E_WORKSPACE       # (the next thing that is looked at)
