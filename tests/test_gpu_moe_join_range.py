"""moe_down in float16: an expert's row may lie past the type's largest number where the weighted sum of a token's rows does not, in a call of any
size."""
import numpy as np
import pytest
import torch

import tritonix
from tritonix_amd.ops import mx

pytestmark = pytest.mark.gpu

INNER, WIDTH, TOP_K, EXPERTS = 256, 1024, 8, 16


def case(device, tokens, seed):
    """Rows and weights of small whole numbers that microscaling keeps, whose products add up without rounding in 32 bits: |row| up to 256 * 4 * 256 = 2^18."""
    g = torch.Generator("cpu").manual_seed(seed)
    pick = lambda values, *s: torch.tensor(values)[torch.randint(0, len(values), s, generator=g)]      # noqa: E731
    h = pick([1.0, 2.0, 3.0, 4.0], tokens * TOP_K, INNER)
    h[:, ::32] = 4.0                                       # every block has the scale 1
    w = pick([64.0, 128.0, 192.0, 256.0], EXPERTS, INNER, WIDTH)
    w[:, ::32] = 256.0
    experts = torch.stack([torch.randperm(EXPERTS, generator=g)[:TOP_K] for _ in range(tokens)])
    weights = pick([1 / 64, 3 / 128, 1 / 32], tokens, TOP_K)
    return h.half().to(device), w, experts.to(device), weights.to(device)


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("tokens", [64, 1300])                             # 2 and 43 MB of rows in 32 bits
def test_rows_past_the_largest_number(device, monkeypatch, tokens, native):
    if not native:
        monkeypatch.setattr(mx, "native", mx._Interpreter)
    h, w, experts, weights = case(device, tokens, 3)
    q = tritonix.mx_quantize(w.to(device), dim=-2)
    r = tritonix.moe_plan(experts, weights, EXPERTS)
    out = tritonix.moe_down(h, q, r).cpu().double().numpy()
    rows, hd, wd, want, largest = r.rows.cpu().numpy(), h.cpu().double().numpy(), w.double().numpy(), np.zeros((tokens, WIDTH)), 0.0
    for e in range(EXPERTS):
        pairs = np.argwhere(experts.cpu().numpy() == e)
        y = hd[rows[pairs[:, 0], pairs[:, 1]]] @ wd[e]
        largest = max(largest, np.abs(y).max())
        want[pairs[:, 0]] += weights.cpu().double().numpy()[pairs[:, 0], pairs[:, 1], None] * y
    assert largest > 65504 > want.max()
    # products and their sums are exact in 32 bits (whole multiples of 2^-1 below 2^17): what is left is the rounding to float16
    np.testing.assert_array_equal(out, torch.from_numpy(want).half().double().numpy())


def test_a_token_is_the_same_in_a_small_batch(device):
    h, w, experts, weights = case(device, 1300, 4)
    q = tritonix.mx_quantize(w.to(device), dim=-2)
    r = tritonix.moe_plan(experts, weights, EXPERTS)
    out = tritonix.moe_down(h, q, r)
    few = tritonix.moe_plan(experts[:5], weights[:5], EXPERTS)
    rows = torch.empty(5 * TOP_K, INNER, dtype=torch.float16, device=device)
    rows[few.rows.flatten().long()] = h[r.rows[:5].flatten().long()]
    assert torch.equal(tritonix.moe_down(rows, q, few), out[:5])
