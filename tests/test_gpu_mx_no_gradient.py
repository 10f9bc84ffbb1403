"""Products that have no derivative say so: differentiating their result is an error where an input asks for its gradient, never a gradient
that silently lacks a term."""
import pytest
import torch

import tritonix
from tritonix_amd.ops import mx

pytestmark = pytest.mark.gpu


def rand(device, *shape, dtype=torch.bfloat16, seed=0):
    return torch.randn(shape, generator=torch.Generator("cpu").manual_seed(seed)).to(dtype).to(device)


def calls(device, tokens):
    """name -> (call, the input that asks for a gradient)"""
    x, w = rand(device, tokens, 64), rand(device, 64, 32, seed=1)
    q = tritonix.mx_quantize(w, dim=0)
    h = rand(device, 2 * tokens, 32, seed=2)
    w12, w3 = (tritonix.mx_quantize(rand(device, *s, seed=3), dim=-2) for s in ((4, 64, 64), (4, 32, 64)))
    r = tritonix.moe_route(rand(device, tokens, 4, dtype=torch.float32, seed=4), 2)
    weighted = lambda v: tritonix.Routing(**{**vars(r), "weights": v})      # noqa: E731
    return {
        "matmul a": (lambda v: tritonix.mx_matmul(v, q), x), "matmul a, other type": (lambda v: tritonix.mx_matmul(v, q, torch.float32), x),
        "matmul b": (lambda v: tritonix.mx_matmul(x, v), w), "matmul b of a quantised a": (lambda v: tritonix.mx_matmul(tritonix.mx_quantize(x), v), w),
        "glu x": (lambda v: tritonix.mx_glu(v, q), x), "glu w": (lambda v: tritonix.mx_glu(x, v), w),
        "moe_glu x": (lambda v: tritonix.moe_glu(v, w12, r), x), "moe_down h": (lambda v: tritonix.moe_down(v, w3, r), h),
        "moe_down weights": (lambda v: tritonix.moe_down(h, w3, weighted(v)), r.weights),
        "moe_down weights, other type": (lambda v: tritonix.moe_down(h, w3, weighted(v), torch.float32), r.weights),
        "moe_ffn x": (lambda v: tritonix.moe_ffn(v, w12, w3, r), x), "moe_ffn weights": (lambda v: tritonix.moe_ffn(x, w12, w3, weighted(v)), r.weights),
    }


NAMES = ["matmul a", "matmul a, other type", "matmul b", "matmul b of a quantised a", "glu x", "glu w", "moe_glu x", "moe_down h", "moe_down weights",
         "moe_down weights, other type", "moe_ffn x", "moe_ffn weights"]


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("tokens", [2, 40])
@pytest.mark.parametrize("native", [True, False])
def test_differentiating_is_an_error(device, monkeypatch, name, tokens, native):
    if not native:
        monkeypatch.setattr(mx, "native", mx._Interpreter)
    call, source = calls(device, tokens)[name]
    want = call(source)
    assert not want.requires_grad
    leaf = source.detach().clone().requires_grad_(True)
    with torch.no_grad():
        assert not call(leaf).requires_grad
    y = call(leaf)
    assert y.dtype == want.dtype and torch.equal(y.detach(), want)
    with pytest.raises(RuntimeError, match="no gradient"):
        (y.float().sum() + leaf.float().sum()).backward()                  # (a term of its own does not hide the missing one)
    with pytest.raises(RuntimeError, match="no gradient"):
        torch.autograd.grad(call(leaf).float().sum(), leaf, allow_unused=True)


def test_the_router_is_not_trained_on_half_of_its_loss(device):
    """The block's loss and a balance term: the weights carry the gradient of the second alone, so the sum cannot be differentiated."""
    x, logits = rand(device, 20, 64), rand(device, 20, 4, dtype=torch.float32, seed=4).requires_grad_(True)
    w12, w3 = (tritonix.mx_quantize(rand(device, *s, seed=3), dim=-2) for s in ((4, 64, 64), (4, 32, 64)))
    r = tritonix.moe_route(logits, 2)
    y = tritonix.moe_ffn(x, w12, w3, r)
    with pytest.raises(RuntimeError, match="no gradient"):
        (y.float().square().mean() + r.weights.square().sum()).backward()
    r = tritonix.moe_route(logits, 2)
    (g,) = torch.autograd.grad(r.weights.square().sum(), logits)          # the balance term by itself
    assert bool((g != 0).any())


def test_the_layer_that_is_trained_still_is(device):
    """mx_linear's products are mx_matmul's on the interpreter's path: no error there."""
    x, w, dy = rand(device, 33, 64).requires_grad_(True), rand(device, 64, 32, seed=1).requires_grad_(True), rand(device, 33, 32, seed=2)
    for native in (mx.find_native(), mx._Interpreter):
        mx.native = native
        try:
            dx, dw = torch.autograd.grad(tritonix.mx_linear(x, w), (x, w), dy)
        finally:
            mx.native = None
        assert bool((dx != 0).any()) and bool((dw != 0).any())
