"""The calls of linear layers, layer normalisation and grouped products that csrc/launch.cpp makes without the interpreter."""
from __future__ import annotations

import ctypes

import torch

from tritonix_amd import _C
from tritonix_amd import kernel as _kernel
from tritonix_amd.kernel import launch_module
from tritonix_amd.ops import mx as _mx

# the module, or what stands in for it where it cannot be used; found with the first call
module = None


def counted_workspace(index: int, stream: int, nbytes: int) -> torch.Tensor:
    """Scratch of products whose K is cut, its counters zero: the stream's own buffer or, for a launch that is recorded into a HIP graph, one
    of the graph's (two graphs of one stream may be replayed on two)."""
    device = torch.device("cuda", index)
    if _kernel._capturing():
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
        ws[:_C.WS_COUNTER_BYTES].zero_()
        return ws
    return _kernel._workspace(device, stream, nbytes)


def find():
    global module
    native = launch_module()
    if native is None:
        module = _mx._Interpreter
    else:
        lib = _C.load()
        native.bind_blocks(tuple(ctypes.cast(fn, ctypes.c_void_p).value for fn in (
            lib.tnx_linear_workspace_bytes, lib.tnx_linear_scratch_bytes, lib.tnx_linear, lib.tnx_linear_gradient_bytes, lib.tnx_linear_gradient,
            lib.tnx_layer_norm, lib.tnx_layer_norm_workspace_bytes, lib.tnx_layer_norm_backward, lib.tnx_grouped, lib.tnx_grouped_workspace_bytes)))
        module = native
    return module
