"""A routing that moe_plan made of a choice from elsewhere is good for the experts' products, and for nothing that it does not know."""
import pytest
import torch

import tritonix

pytestmark = pytest.mark.gpu


def rand(device, *shape, dtype=torch.float32, seed=0):
    return torch.randn(shape, generator=torch.Generator("cpu").manual_seed(seed)).to(dtype).to(device)


def test_a_choice_made_elsewhere_has_no_gradient_of_logits(device):
    """moe_plan knows neither scores nor scale, so the gradient of logits cannot be answered from its routing."""
    logits = rand(device, 9, 8)
    made = tritonix.moe_route(logits, 2, scoring="sigmoid", scale=2.5)
    plan = tritonix.moe_plan(made.experts, made.weights, 8)
    with pytest.raises(ValueError, match="moe_plan"):
        tritonix.moe_route_backward(torch.ones(9, 2, device=device), logits, plan)
    assert tritonix.moe_route_backward(torch.ones(9, 2, device=device), logits, made).shape == (9, 8)
    w12, w3 = (tritonix.mx_quantize(rand(device, *s), dim=-2) for s in ((8, 64, 64), (8, 32, 64)))
    x = rand(device, 9, 64, dtype=torch.bfloat16)
    assert torch.equal(tritonix.moe_ffn(x, w12, w3, plan), tritonix.moe_ffn(x, w12, w3, made))
