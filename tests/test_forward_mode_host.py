"""Forward-mode derivatives are refused, by every operator that has gradients or says that it has none, before anything is looked for on a device."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import tritonix

BF16, F32 = torch.bfloat16, torch.float32


def t(*shape, dtype=F32):
    return torch.ones(shape, dtype=dtype)


CALLS = {
    "linear": (lambda x, w, b, r: tritonix.linear(x, w, b, "silu", r), ((4, 16), (16, 32), (32,), (4, 32))),
    "linear of three dimensions": (lambda x, w, b, r: tritonix.linear(x, w, b, None, r), ((2, 4, 16), (16, 32), (32,), (2, 4, 32))),
    "layer_norm": (lambda x, w, b: tritonix.layer_norm(x, w, b), ((4, 16), (16,), (16,))),
    "layer_norm of three dimensions": (lambda x: tritonix.layer_norm(x), ((2, 4, 16),)),
    "grouped_matmul": (lambda x, w: tritonix.grouped_matmul(x, w, torch.tensor([0, 2, 4], dtype=torch.int32)), ((4, 16), (2, 16, 32))),
    "mx_quantize": (lambda x: tritonix.mx_quantize(x, -1), ((4, 256),)),
    "moe_route": (lambda x: tritonix.moe_route(x, 2), ((4, 8),)),
}


@pytest.mark.parametrize("call", list(CALLS))
def test_a_tangent_is_refused(call):
    f, shapes = CALLS[call]
    for i in range(len(shapes)):
        with forward_ad.dual_level():
            given = [t(*s) for s in shapes]
            with pytest.raises(ValueError, match="HIP device"):
                f(*given)
            given[i] = forward_ad.make_dual(given[i], t(*shapes[i]))
            with pytest.raises(RuntimeError, match="forward"):
                f(*given)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward"):
                f(*given)
    # what is left of a tangent after its level is an ordinary tensor
    with pytest.raises(ValueError, match="HIP device"):
        f(*given)
