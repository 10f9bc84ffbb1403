"""Routing where scores are close to nothing, and softmax scores under a bias."""
import math

import numpy as np
import pytest
import torch

import tritonix
from tests import mx_reference as ref
from tests.test_gpu_moe import REL, check_route, formula_gradient, separated

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [3, 1500])
@pytest.mark.parametrize("experts,k", [(8, 1), (60, 6), (256, 8)])
@pytest.mark.parametrize("depth", [-80.0, -87.9, -88.3, -88.6, -95.0])
def test_sigmoid_scores_next_to_nothing(device, tokens, experts, k, depth):
    """Equal scores down to the smallest numbers of 32 bits: a share is 1 / k of the scale, or, where the scores are zero in 32 bits, zero.  Never an
    infinity or NaN, and neither in the gradient, whose share of equal scores is scale / k (g - mean g) (1 - s)."""
    logits, grad = torch.full((tokens, experts), depth, device=device), torch.randn(tokens, k, generator=torch.Generator("cpu").manual_seed(1)).to(device)
    r = tritonix.moe_route(logits, k, scoring="sigmoid", scale=2.5)
    assert bool((r.experts == torch.arange(k, device=device)).all())
    got = tritonix.moe_route_backward(grad, logits, r)
    if bool((r.weights == 0).all()):
        assert depth < -88 and bool((got == 0).all())
        return
    # (a subnormal score has 21 bits here, and so have shares of it)
    np.testing.assert_allclose(r.weights.cpu().double().numpy(), 2.5 / k, rtol=2.0 ** -18)
    want = 2.5 / k * (grad.double() - grad.double().mean(dim=1, keepdim=True))
    assert float((got[:, :k].double() - want).abs().max()) <= 2.0 ** -16 * 2.5 * float(grad.abs().max()) and bool((got[:, k:] == 0).all())


@pytest.mark.parametrize("tokens", [3, 1500])
@pytest.mark.parametrize("depth", [-20.0, -80.0, -87.0, -89.0, -95.0, -103.0, -200.0])
@pytest.mark.parametrize("renormalize", [True, False])
def test_softmax_scores_next_to_nothing(device, tokens, depth, renormalize):
    """A bias that chooses experts far below the row's largest: their shares are a softmax among themselves however small they are."""
    experts, k = 40, 5
    logits = separated(tokens, experts, torch.float32, 5) + depth
    logits[:, 7] = 0.0
    bias = torch.zeros(experts)
    bias[7] = -10.0
    bias[11:11 + k] = 5.0
    r = tritonix.moe_route(logits.to(device), k, bias=bias.to(device), renormalize=renormalize, scale=2.5)
    assert torch.equal(r.experts.cpu().sort(dim=1).values.long(), torch.arange(11, 11 + k).expand(tokens, k))
    x = logits.double()
    score = torch.softmax(x.gather(1, r.experts.cpu().long()) if renormalize else x, dim=1)
    want = 2.5 * (score if renormalize else score.gather(1, r.experts.cpu().long()))
    # (an exponential of an argument up to 2^7, where it is no subnormal number)
    np.testing.assert_allclose(r.weights.cpu().double().numpy(), want.numpy(), rtol=REL * 4, atol=2.0 ** -126)


@pytest.mark.parametrize("experts,k,groups,top,group_top", [(8, 2, 1, 1, 1), (64, 6, 8, 4, 2), (60, 4, 4, 1, 1), (256, 8, 8, 4, 2), (512, 9, 1, 1, 1), (1024, 32, 2, 1, 1)])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("tokens", [4, 60, 1100])
def test_softmax_under_a_bias(device, experts, k, groups, top, group_top, renormalize, tokens):
    """Choice, weights and the gradient of the logits against the definition; rows whose keys, or groups, lie within the error of 32-bit scores left out."""
    logits = separated(tokens, experts, torch.float32, groups)
    bias = (torch.randn(experts, generator=torch.Generator("cpu").manual_seed(experts)) * 0.05).float()
    keys = torch.softmax(logits.double(), dim=1) + bias.double()
    near = (keys.sort(dim=1).values.diff(dim=1) < 1e-7).any(dim=1)
    worth = keys.view(tokens, groups, -1).topk(min(group_top, experts // groups), dim=-1).values.sum(-1).sort(dim=1).values
    near |= (worth.diff(dim=1) < 1e-7).any(dim=1)
    logits = logits[~near]
    assert len(logits) >= tokens // 4
    options = dict(num_groups=groups, top_groups=top, group_top=group_top, renormalize=renormalize, scale=1.5)
    r = check_route(device, logits, k, bias=bias, **options)
    grad = torch.randn(len(logits), k, generator=torch.Generator("cpu").manual_seed(1))
    got = tritonix.moe_route_backward(grad.to(device), logits.to(device), r).cpu().double()
    want = formula_gradient(logits, grad, r.experts.cpu(), "softmax", renormalize, 1.5)
    assert float((got - want).abs().max()) <= REL * 8 * 1.5 * float(grad.abs().max()) * float(r.weights.max())


def test_shares_of_rows_with_masked_experts(device):
    """-inf and the type's lowest value among the chosen of a biased softmax."""
    logits = separated(6, 16, torch.float32, 3)
    logits[0, 2:] = -math.inf
    logits[1, 3:] = torch.finfo(torch.float32).min
    logits[2] = -math.inf
    bias = torch.linspace(0.0, 0.1, 16)
    for renormalize in (True, False):
        r = tritonix.moe_route(logits.to(device), 4, bias=bias.to(device), renormalize=renormalize)
        weights, experts = ref.route(logits, 4, bias=bias, renormalize=renormalize)
        np.testing.assert_array_equal(r.experts.cpu().numpy(), experts)
        np.testing.assert_allclose(r.weights.cpu().double().numpy(), weights, rtol=REL, atol=2.0 ** -126)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("tokens", [2, 1100])
def test_the_lowest_value_is_no_score(device, dtype, scoring, tokens):
    """Experts masked by the type's lowest value that a bias chooses all the same: weight zero, alone and beside one that has a score."""
    logits = separated(tokens, 16, torch.float32, 3).to(dtype)
    logits[:, 8:] = torch.finfo(dtype).min
    bias = torch.zeros(16)
    bias[8:12] = 3.0
    check_route(device, logits, 4, scoring=scoring, bias=bias)
    r = check_route(device, logits, 5, scoring=scoring, bias=bias)
    assert bool((r.weights[:, :4] == 0).all()) and bool((r.weights[:, 4] == 1).all())
