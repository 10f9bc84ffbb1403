"""Routing and the experts' products on the GPU against row-by-row definitions in 64 bits."""
import math

import numpy as np
import pytest
import torch

import tritonix
from tests import mx_reference as ref

pytestmark = pytest.mark.gpu

# Scores, sums over at most 1024 of them and quotients in 32 bits, exponentials good to a few units: 2^-18 covers 1024 additions' rounding (the sum's terms
# are positive, so its relative error is below 10 roundings of a tree) with room for the exponential of an argument up to 2^5
REL = 2.0 ** -18


def separated(tokens, experts, dtype, seed):
    """Rows whose values are a shuffled grid: no two scores (nor biased scores with a bias of this grid's spacing) are close."""
    g = torch.Generator("cpu").manual_seed(seed)
    grid = torch.linspace(-2.0, 2.0, experts).to(dtype)
    assert len(set(grid.tolist())) == experts
    return torch.stack([grid[torch.randperm(experts, generator=g)] for _ in range(tokens)])


def check_route(device, logits, k, **options):
    bias = options.get("bias")
    r = tritonix.moe_route(logits.to(device), k, **{**options, "bias": bias.to(device) if bias is not None else None})
    weights, experts = ref.route(logits, k, **options)
    np.testing.assert_array_equal(r.experts.cpu().numpy(), experts)
    np.testing.assert_allclose(r.weights.cpu().double().numpy(), weights, rtol=REL, atol=2.0 ** -126)
    offsets, order, rows = ref.plan(r.experts.cpu(), logits.shape[1])
    assert r.offsets.cpu().tolist() == offsets and r.order.cpu().tolist() == order and r.rows.cpu().reshape(-1).tolist() == rows
    return r


@pytest.mark.parametrize("experts,k", [(1, 1), (2, 2), (7, 3), (8, 8), (32, 4), (33, 2), (64, 6), (100, 32), (128, 8), (129, 5), (256, 8), (300, 10),
                                       (512, 4), (513, 9), (1024, 32)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("tokens", [1, 5, 70])
def test_choice_and_plan(device, experts, k, scoring, tokens):
    for renormalize, scale in ((True, 1.0), (False, 2.5)):
        check_route(device, separated(tokens, experts, torch.float32, experts + tokens), k, scoring=scoring, renormalize=renormalize, scale=scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_sixteen_bit_logits_with_ties(device, dtype):
    g = torch.Generator("cpu").manual_seed(3)
    logits = (torch.randint(-8, 8, (300, 40), generator=g) / 4).to(dtype)      # many equal logits: the lower expert goes first
    check_route(device, logits, 6)
    check_route(device, torch.zeros(9, 64, dtype=dtype), 8, scoring="sigmoid")


@pytest.mark.parametrize("experts,groups,top", [(8, 4, 2), (64, 8, 4), (60, 4, 1), (256, 8, 4), (512, 64, 3), (1024, 2, 1)])
@pytest.mark.parametrize("group_top", [1, 2])
def test_biased_choice_within_groups(device, experts, groups, top, group_top):
    tokens = 40
    logits = separated(tokens, experts, torch.float32, groups)
    g = torch.Generator("cpu").manual_seed(experts)
    bias = (torch.randn(experts, generator=g) * 0.1).float()
    # rows in which two keys, or two groups, lie within the error of 32-bit scores have no one answer: left out
    s = torch.sigmoid(logits.double()) + bias.double()
    near = (s.sort(dim=1).values.diff(dim=1) < 1e-6).any(dim=1)
    worth = s.view(tokens, groups, -1).topk(min(group_top, experts // groups), dim=-1).values.sum(-1).sort(dim=1).values
    near |= (worth.diff(dim=1) < 1e-6).any(dim=1)
    assert int((~near).sum()) >= 8
    k = min(8, experts // groups * top)
    check_route(device, logits[~near], k, scoring="sigmoid", bias=bias, num_groups=groups, top_groups=top, group_top=group_top, scale=2.5)


def test_groups_without_a_bias(device):
    check_route(device, separated(33, 64, torch.float32, 9), 4, num_groups=8, top_groups=2)
    check_route(device, separated(33, 64, torch.float32, 9), 4, num_groups=8, top_groups=8)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_masked_rows_and_values_that_are_not_numbers(device, scoring):
    x = separated(12, 24, torch.float32, 4)
    x[0] = -math.inf                                      # nothing to choose
    x[1, 3:] = -math.inf                                  # three experts for five slots
    x[2] = torch.finfo(torch.float32).min                 # the type's lowest value is a number: all equal
    x[3, 1:] = torch.finfo(torch.float32).min
    x[4, 7] = math.nan
    x[5, 7] = math.inf
    x[6, ::2] = -math.inf
    x[7] = 1e30 * x[7]
    check_route(device, x, 5, scoring=scoring)
    check_route(device, x, 5, scoring=scoring, renormalize=False)
    bias = torch.zeros(24)
    bias[2], bias[5] = -math.inf, math.nan                # never chosen
    if scoring == "sigmoid":
        r = tritonix.moe_route(x.to(device), 5, scoring=scoring, bias=bias.to(device))
        assert not bool(((r.experts == 2) | (r.experts == 5)).any())


def test_strided_logits(device):
    base = separated(50, 96, torch.float32, 8)
    check_route(device, base[:, :40], 4)
    check_route(device, base[::3, 7:], 4)
    check_route(device, base.t(), 3)


@pytest.mark.parametrize("tokens,k,experts", [(1, 1, 1), (0, 2, 8), (512, 1, 5), (513, 1, 5), (64, 8, 16), (65, 8, 16), (3000, 6, 60), (20000, 8, 128), (1500, 4, 1024)])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64], ids=str)
def test_plan_of_given_experts(device, tokens, k, experts, dtype):
    g = torch.Generator("cpu").manual_seed(tokens)
    e = torch.randint(-2, experts + 2, (tokens, k), generator=g).to(dtype)      # empty slots, and the same expert twice in a row
    r = tritonix.moe_plan(e.to(device), torch.ones(tokens, k, device=device), experts)
    flat = torch.where((e >= 0) & (e < experts), e, experts).reshape(-1)
    order = torch.sort(flat, stable=True).indices
    total = int((flat < experts).sum())
    counts = torch.bincount(flat, minlength=experts + 1)[:experts]
    assert r.offsets.cpu().tolist() == [0] + counts.cumsum(0).tolist()
    assert torch.equal(r.order.cpu()[:total].long(), order[:total]) and bool((r.order.cpu()[total:] == -1).all())
    rows = torch.full((tokens * k,), -1)
    rows[order[:total]] = torch.arange(total)
    assert torch.equal(r.rows.cpu().reshape(-1).long(), rows)


def formula_gradient(logits, grad, experts, scoring, renormalize, scale):
    x = logits.double().cpu().clone().requires_grad_(True)
    s = torch.softmax(x, dim=1) if scoring == "softmax" else torch.sigmoid(x)
    chosen = experts >= 0
    w = torch.gather(s, 1, experts.clamp(min=0).long()) * chosen
    if renormalize:
        w = w / w.sum(dim=1, keepdim=True)
    (out,) = torch.autograd.grad((w * scale * grad.double().cpu()).sum(), x)
    return out


@pytest.mark.parametrize("experts,k", [(2, 1), (8, 8), (33, 4), (64, 6), (128, 8), (200, 20), (500, 9), (1000, 32)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_gradient_is_the_formula(device, experts, k, scoring, renormalize):
    tokens = 37
    logits = separated(tokens, experts, torch.float32, k)
    grad = torch.randn(tokens, k, generator=torch.Generator("cpu").manual_seed(1))
    x = logits.to(device).requires_grad_(True)
    r = tritonix.moe_route(x, k, scoring=scoring, renormalize=renormalize, scale=1.5)
    (got,) = torch.autograd.grad(r.weights, x, grad.to(device))
    want = formula_gradient(logits, grad, r.experts.cpu(), scoring, renormalize, 1.5)
    # differences of terms up to |grad| * weight: the error is relative to those
    top = 1.5 * grad.abs().max().double() * r.weights.detach().cpu().double().max()
    assert float((got.cpu().double() - want).abs().max()) <= REL * 8 * float(top)
    again = tritonix.moe_route_backward(grad.to(device), logits.to(device), r)
    assert torch.equal(again, got)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_gradient_is_the_differences(device, scoring, renormalize):
    """Central differences of the forward pass, h = 2^-6: their third-order term is below h^2 / 6 of the weights' third derivative (below 1), 4e-5; rounding
    adds 2^-22 / h = 2e-5 for each of k terms."""
    logits = separated(4, 12, torch.float32, 2)           # neighbours 0.36 apart: the choice does not change within h
    grad = torch.randn(4, 3, generator=torch.Generator("cpu").manual_seed(1))
    run = lambda x: tritonix.moe_route(x.to(device), 3, scoring=scoring, renormalize=renormalize)      # noqa: E731
    got = tritonix.moe_route_backward(grad.to(device), logits.to(device), run(logits)).cpu()
    h = 2.0 ** -6
    for e in range(12):
        up, down = logits.clone(), logits.clone()
        up[:, e] += h
        down[:, e] -= h
        diff = ((run(up).weights - run(down).weights).cpu() * grad).sum(dim=1) / (2 * h)
        assert float((diff - got[:, e]).abs().max()) <= 1e-3


def test_gradient_of_masked_rows(device):
    logits = separated(6, 16, torch.float32, 3)
    logits[0] = -math.inf
    logits[1, 2:] = -math.inf
    logits[2, 5] = math.nan
    grad = torch.ones(6, 4)
    grad[1, 0] = 3.0
    for scoring in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            r = tritonix.moe_route(logits.to(device), 4, scoring=scoring, renormalize=renormalize)
            got = tritonix.moe_route_backward(grad.to(device), logits.to(device), r).cpu()
            assert bool((got[0] == 0).all()) and bool((got[1, 2:] == 0).all()) and bool(torch.isnan(got[2]).all())
            assert bool(torch.isfinite(got[[0, 1, 3, 4, 5]]).all())
            assert bool((got[1, :2] != 0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_gradient_in_sixteen_bits(device, dtype):
    logits = separated(20, 16, dtype, 3)
    grad = torch.randn(20, 4, generator=torch.Generator("cpu").manual_seed(1))
    r = tritonix.moe_route(logits.to(device), 4, renormalize=False)
    got = tritonix.moe_route_backward(grad.to(device), logits.to(device), r)
    want = formula_gradient(logits, grad, r.experts.cpu(), "softmax", False, 1.0).numpy()
    assert got.dtype == dtype
    tol = REL * 8 * float(grad.abs().max()) + ref.rounding(want, dtype)
    assert (np.abs(got.cpu().double().numpy() - want) <= tol).all()


def expert_case(tokens, experts, k, d, f, seed, holes=0.0, skew=False):
    g = torch.Generator("cpu").manual_seed(seed)
    x = torch.randn(tokens, d, generator=g).bfloat16()
    w12 = (torch.randn(experts, d, 2 * f, generator=g) / math.sqrt(d)).bfloat16()
    w3 = (torch.randn(experts, f, d, generator=g) / math.sqrt(f)).bfloat16()
    if skew:                                              # every token to the last expert first
        e = torch.full((tokens, k), experts - 1)
        e[:, 1:] = torch.randint(0, experts, (tokens, k - 1), generator=g)
    else:
        e = torch.stack([torch.randperm(experts, generator=g)[:k] for _ in range(tokens)]) if tokens else torch.zeros(0, k, dtype=torch.long)
    e = torch.where(torch.rand(e.shape, generator=g) < holes, torch.full_like(e, -1), e)
    weights = torch.rand(e.shape, generator=g)
    return x, w12, w3, e, weights


CASES = [(1, 8, 2, 64, 32, 0.0, False), (1, 64, 8, 512, 300, 0.0, False), (3, 5, 2, 33, 17, 0.0, False), (40, 8, 3, 100, 65, 0.2, False),
         (70, 100, 4, 96, 40, 0.0, False), (200, 4, 2, 300, 130, 0.1, False), (90, 6, 2, 260, 64, 0.0, True), (300, 3, 2, 128, 200, 0.0, True),
         (600, 2, 1, 200, 300, 0.5, False), (1500, 6, 4, 256, 520, 0.0, False), (10, 3, 2, 64, 32, 1.0, False), (700, 70, 2, 130, 64, 0.0, True), (2100, 5, 4, 1030, 64, 0.1, False)]


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_experts_products(device, case, dtype):
    tokens, experts, k, d, f, holes, skew = case
    x, w12, w3, e, weights = expert_case(tokens, experts, k, d, f, tokens + d, holes, skew)
    r = tritonix.moe_plan(e.to(device), weights.to(device), experts)
    q12, q3 = tritonix.mx_quantize(w12.to(device), dim=-2), tritonix.mx_quantize(w3.to(device), dim=-2)
    xv, w12v, w3v = ref.values(x), ref.values(w12, -2), ref.values(w3, -2)
    offsets, order = r.offsets.cpu().tolist(), r.order.cpu().tolist()

    h = tritonix.moe_glu(x.to(device), q12, r, out_dtype=dtype)
    got = h.cpu().double().numpy()
    assert got.shape == (tokens * k, f)
    assert (got[offsets[-1]:] == 0).all()
    for i in range(experts):
        lo, hi = offsets[i], offsets[i + 1]
        a = xv[[p // k for p in order[lo:hi]]]
        want, tol = ref.gated(a @ w12v[i], ref.product_bound(a, w12v[i], d), "silu")
        assert (np.abs(got[lo:hi] - want) <= tol + ref.rounding(np.abs(want) + tol, dtype)).all(), i

    hin = torch.randn(tokens * k, f, generator=torch.Generator("cpu").manual_seed(9)).bfloat16()
    out = tritonix.moe_down(hin.to(device), q3, r, out_dtype=dtype).cpu().double().numpy()
    hv = ref.values(hin)
    want, tol = np.zeros((tokens, d)), np.zeros((tokens, d))
    for i in range(experts):
        lo, hi = offsets[i], offsets[i + 1]
        y = hv[lo:hi] @ w3v[i]
        t = ref.product_bound(hv[lo:hi], w3v[i], f)
        t = t + ref.rounding(np.abs(y) + t, torch.float32 if tokens * k * d * 4 <= 32 << 20 else dtype)
        for row, p in enumerate(order[lo:hi]):
            w = float(weights.reshape(-1)[p])
            want[p // k] += w * y[row]
            tol[p // k] += w * t[row] + 2.0 ** -22 * k * w * (np.abs(y[row]) + t[row])
    assert (np.abs(out - want) <= tol + ref.rounding(np.abs(want) + tol, dtype)).all()


def test_feed_forward_block_is_its_parts_and_any_stream(device):
    x, w12, w3, e, weights = expert_case(50, 8, 2, 128, 96, 1)
    logits = separated(50, 8, torch.float32, 1).to(device)
    q12, q3 = tritonix.mx_quantize(w12.to(device), dim=-2), tritonix.mx_quantize(w3.to(device), dim=-2)
    x = x.to(device)
    r = tritonix.moe_route(logits, 2)
    y = tritonix.moe_ffn(x, q12, q3, r)
    assert torch.equal(y, tritonix.moe_down(tritonix.moe_glu(tritonix.mx_quantize(x), q12, r), q3, r))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = tritonix.moe_ffn(x, q12, q3, tritonix.moe_route(logits, 2))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, again)


def test_graph_of_a_block_replays(device):
    x, w12, w3, e, weights = expert_case(6, 16, 4, 256, 128, 1)
    q12, q3 = tritonix.mx_quantize(w12.to(device), dim=-2), tritonix.mx_quantize(w3.to(device), dim=-2)
    x, logits = x.to(device), separated(6, 16, torch.float32, 1).to(device)
    step = lambda: tritonix.moe_ffn(x, q12, q3, tritonix.moe_route(logits, 4))      # noqa: E731
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        logits.copy_(separated(6, 16, torch.float32, 20 + i))
        x.copy_(torch.randn(6, 256, generator=torch.Generator("cpu").manual_seed(i)).bfloat16())
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_no_tokens(device):
    x, w12, w3, e, weights = expert_case(1, 4, 2, 64, 32, 1)
    q12, q3 = tritonix.mx_quantize(w12.to(device), dim=-2), tritonix.mx_quantize(w3.to(device), dim=-2)
    r = tritonix.moe_route(torch.zeros(0, 4, device=device), 2)
    assert r.offsets.cpu().tolist() == [0] * 5
    assert tritonix.moe_ffn(x[:0].to(device), q12, q3, r).shape == (0, 64)
