"""The routed block of examples/routed_ffn.py: what a replayed graph answers is what the eager call answers, token for token, and both are the definition's."""
import os
import runpy

import numpy as np
import pytest
import torch

import tritonix
from tests import mx_reference as ref

pytestmark = pytest.mark.gpu

WIDTH, INNER, EXPERTS, TOP_K = 256, 128, 8, 2


@pytest.fixture(scope="module")
def block():
    return runpy.run_path(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "routed_ffn.py"))["block"]


def tensors(device, tokens):
    g = torch.Generator("cpu").manual_seed(5)
    rand = lambda *s: torch.randn(s, generator=g)      # noqa: E731
    return (rand(tokens, WIDTH).bfloat16().to(device), (rand(WIDTH, EXPERTS) / WIDTH ** 0.5).bfloat16().to(device),
            (rand(EXPERTS, WIDTH, 2 * INNER) / WIDTH ** 0.5).bfloat16(), (rand(EXPERTS, INNER, WIDTH) / INNER ** 0.5).bfloat16())


@pytest.mark.parametrize("tokens", [1, 3, 40])
def test_replays_are_the_eager_call(device, block, tokens):
    x, w_router, w12, w3 = tensors(device, 6 * tokens)
    q12, q3 = tritonix.mx_quantize(w12.to(device), dim=-2), tritonix.mx_quantize(w3.to(device), dim=-2)
    given = x[:tokens].clone()
    with torch.no_grad():
        block(given, w_router, q12, q3, TOP_K)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, routing = block(given, w_router, q12, q3, TOP_K)
        answers = []
        for i in range(6):
            given.copy_(x[i * tokens:(i + 1) * tokens])
            want, eager = block(given.clone(), w_router, q12, q3, TOP_K)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(routing.experts, eager.experts) and torch.equal(routing.weights, eager.weights)
            answers.append(out.clone())
    assert all(not torch.equal(a, b) for a, b in zip(answers, answers[1:]))


@pytest.mark.parametrize("tokens", [1, 40])
def test_the_block_is_the_definition(device, block, tokens):
    """Each stage from the one before it as the library left it: a code of the intermediate turns on its last bit, so the bound cannot pass through."""
    x, w_router, w12, w3 = tensors(device, tokens)
    q12, q3 = tritonix.mx_quantize(w12.to(device), dim=-2), tritonix.mx_quantize(w3.to(device), dim=-2)
    with torch.no_grad():
        y, r = block(x, w_router, q12, q3, TOP_K)
        logits, h = tritonix.mx_linear(x, w_router), tritonix.moe_glu(x, q12, r)
    want = ref.values(x) @ ref.values(w_router, -2)
    tol = ref.product_bound(ref.values(x), ref.values(w_router, -2), WIDTH)
    assert (np.abs(logits.cpu().double().numpy() - want) <= tol + ref.rounding(np.abs(want) + tol, torch.bfloat16)).all()
    weights, experts = ref.route(logits.float(), TOP_K)
    np.testing.assert_array_equal(r.experts.cpu().numpy(), experts)
    np.testing.assert_allclose(r.weights.cpu().double().numpy(), weights, rtol=2.0 ** -18)
    xv, w12v, hv, w3v, rows = ref.values(x), ref.values(w12, -2), ref.values(h), ref.values(w3, -2), r.rows.cpu().numpy()
    hd, yd = h.cpu().double().numpy(), y.cpu().double().numpy()
    for t in range(tokens):
        joined, slack = np.zeros(WIDTH), np.zeros(WIDTH)
        for j in range(TOP_K):
            e, row, weight = experts[t, j], rows[t, j], weights[t, j]
            want, tol = ref.gated(xv[t:t + 1] @ w12v[e], ref.product_bound(xv[t:t + 1], w12v[e], WIDTH), "silu")
            assert (np.abs(hd[row] - want[0]) <= (tol + ref.rounding(np.abs(want) + tol, torch.bfloat16))[0]).all()
            z, dz = hv[row] @ w3v[e], ref.product_bound(hv[row:row + 1], w3v[e], INNER)[0]
            joined += weight * z
            slack += weight * (dz + 2.0 ** -17 * (np.abs(z) + dz))        # (the weight's error, and the sum's in 32 bits)
        assert (np.abs(yd[t] - joined) <= slack + ref.rounding(np.abs(joined) + slack, torch.bfloat16)).all()
