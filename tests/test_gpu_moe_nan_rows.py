"""A token whose router has failed stays visible: NaN weights without an expert reach the block's output, of that token alone."""
import math

import pytest
import torch

import tritonix
from tritonix_amd.ops import mx

pytestmark = pytest.mark.gpu


def rand(device, *shape, dtype=torch.bfloat16, seed=0):
    return torch.randn(shape, generator=torch.Generator("cpu").manual_seed(seed)).to(dtype).to(device)


@pytest.mark.parametrize("tokens", [3, 6, 300])
@pytest.mark.parametrize("width", [33, 2100], ids=["odd", "wide"])
@pytest.mark.parametrize("scoring,bad", [("softmax", math.nan), ("softmax", math.inf), ("sigmoid", math.nan)])
@pytest.mark.parametrize("native", [True, False])
def test_a_row_that_is_not_a_number(device, monkeypatch, tokens, width, scoring, bad, native):
    if not native:
        monkeypatch.setattr(mx, "native", mx._Interpreter)
    x, logits = rand(device, tokens, 64), rand(device, tokens, 8, dtype=torch.float32, seed=1)
    w12, w3 = (tritonix.mx_quantize(rand(device, *s, seed=2), dim=-2) for s in ((8, 64, 96), (8, 48, width)))
    clean = tritonix.moe_ffn(x, w12, w3, tritonix.moe_route(logits, 2, scoring=scoring))
    logits[1, 5] = bad
    r = tritonix.moe_route(logits, 2, scoring=scoring)
    assert r.experts[1].tolist() == [-1, -1]
    for out_dtype in (None, torch.float32):
        y = tritonix.moe_ffn(x, w12, w3, r, out_dtype=out_dtype)
        others = [t for t in range(tokens) if t != 1]
        assert bool(torch.isnan(y[1]).all()) and bool(torch.isfinite(y[others]).all())
        if out_dtype is None:
            assert torch.equal(y[others], clean[others])


def test_empty_slots_are_left_out(device):
    """Of a choice made elsewhere: whatever number an empty slot's weight is, but NaN, it counts for nothing."""
    h, w3 = rand(device, 12, 48), tritonix.mx_quantize(rand(device, 4, 48, 70, seed=2), dim=-2)
    experts = torch.tensor([[0, 1, 2], [3, -1, 0], [-1, 7, -1], [2, -1, 1]], device=device)
    weights = torch.rand(4, 3, generator=torch.Generator("cpu").manual_seed(3)).to(device)
    want = tritonix.moe_down(h, w3, tritonix.moe_plan(experts, weights.masked_fill((experts < 0) | (experts > 3), 0.0), 4))
    for value in (1.0, -math.inf):
        got = tritonix.moe_down(h, w3, tritonix.moe_plan(experts, weights.masked_fill((experts < 0) | (experts > 3), value), 4))
        assert torch.equal(got, want) and bool((got[2] == 0).all())
    weights[1, 1] = math.nan
    got = tritonix.moe_down(h, w3, tritonix.moe_plan(experts, weights, 4))
    assert bool(torch.isnan(got[1]).all()) and torch.equal(got[[0, 2, 3]], want[[0, 2, 3]])
