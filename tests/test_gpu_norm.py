"""Layer normalisation against the definition in 64 bits: values and gradients, rows of one element to rows longer than the registers hold."""
import pytest
import torch

import blocks_reference as ref
import tritonix

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def step(x, weight, bias, dy, eps=1e-5):
    leaves = {"x": x, "weight": weight, "bias": bias}
    leaves = {name: t.detach().requires_grad_(True) for name, t in leaves.items() if t is not None}
    y = tritonix.layer_norm(leaves["x"], leaves.get("weight"), leaves.get("bias"), eps=eps)
    return {"y": y.detach(), **{"d" + name: g for name, g in zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy))}}


def compare(got, want, types):
    assert set(got) == set(want)
    for name in got:
        ref.check(name, got[name], want[name], types.get(name))


# (the last sizes of each kernel's range and the first of the next, both in 16 and in 32 bits)
WIDTHS = [1, 2, 7, 8, 9, 31, 32, 33, 63, 64, 65, 127, 128, 129, 130, 255, 256, 257, 500, 512, 513, 1023, 1024, 1025, 1501, 2048, 2056, 4095, 4096, 4104, 8192, 8200, 16384, 16385, 32768, 32769, 40000]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", WIDTHS)
def test_values_and_gradients(device, dtype, n):
    rows = 5 if n > 4000 else 37
    x = ref.draw(device, rows, n, dtype=dtype, seed=n) * 2 + 0.5
    weight, bias, dy = (ref.draw(device, *s, dtype=dtype, seed=n + i) for i, s in enumerate(((n,), (n,), (rows, n)), 1))
    for w, b in ((weight, bias), (None, None), (weight.float(), None), (None, bias.float())):
        types = {"y": dtype, "dx": dtype, "dweight": None if w is None else w.dtype, "dbias": None if b is None else b.dtype}
        compare(step(x, w, b, dy), ref.layer_norm(x, w, b, 1e-5, dy), types)
        assert torch.equal(tritonix.layer_norm(x, w, b), step(x, w, b, dy)["y"])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n", [(1, 1024), (3, 40), (600, 96), (2050, 130), (5000, 8), (4099, 61), (3001, 100), (2500, 250), (1500, 2050), (700, 16400)])
def test_many_rows(device, dtype, rows, n):
    x, weight, bias, dy = (ref.draw(device, *s, dtype=dtype, seed=i) for i, s in enumerate(((rows, n), (n,), (n,), (rows, n))))
    types = {name: dtype for name in ("y", "dx", "dweight", "dbias")}
    got = step(x, weight, bias, dy)
    compare(got, ref.layer_norm(x, weight, bias, 1e-5, dy), types)
    again = step(x, weight, bias, dy)
    for name in got:
        assert torch.equal(got[name], again[name]), name


def test_a_mean_far_from_zero(device):
    """Variance from centred values: a mean of 1000 standard deviations costs what the mean's own rounding does."""
    x = ref.draw(device, 20, 3000, dtype=torch.float32, seed=1) + 1000.0
    ref.check("y", tritonix.layer_norm(x), ref.layer_norm(x)["y"])


def test_constant_rows(device):
    x = torch.full((3, 100), 7.0, device=device)
    assert torch.equal(tritonix.layer_norm(x), torch.zeros_like(x))
    g = step(x, None, None, ref.draw(device, 3, 100, dtype=torch.float32))
    ref.check("dx", g["dx"], ref.layer_norm(x, dy=ref.draw(device, 3, 100, dtype=torch.float32))["dx"])


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(device, dtype):
    big = ref.draw(device, 60, 400, dtype=dtype, seed=1)
    g0, w0 = ref.draw(device, 60, 400, dtype=dtype, seed=2), ref.draw(device, 400, dtype=dtype, seed=3)
    n = 101
    for name, cut in {"pitch": lambda t: t[:50, 3:3 + n], "every other row": lambda t: t[::2, :n], "every other column": lambda t: t[:40, :2 * n:2], "columns": lambda t: t[:40, :50].t(), "one row for all": lambda t: t[:1, :n].expand(9, n), "reversed": lambda t: t[:, :n].flip(1)}.items():
        x, dy = cut(big), cut(g0)
        w = w0[: 2 * x.shape[1]: 2]
        compare(step(x, w, w, dy), ref.layer_norm(x, w, w, 1e-5, dy), {})
    y = tritonix.layer_norm(big.view(3, 20, 400), w0)
    assert y.shape == (3, 20, 400) and torch.equal(y.view(60, 400), tritonix.layer_norm(big, w0))
    one = tritonix.layer_norm(big[0], w0)
    assert one.shape == (400,) and torch.equal(one, y[0, 0])


def test_numbers_that_are_none(device):
    """A row with a NaN or an infinity is NaN, the others are what they were."""
    x = ref.draw(device, 40, 300, dtype=torch.float32)
    clean = tritonix.layer_norm(x)
    x[4, 7], x[9, 0] = float("nan"), float("-inf")
    y = tritonix.layer_norm(x)
    keep = [i for i in range(40) if i not in (4, 9)]
    assert y[4].isnan().all() and y[9].isnan().all() and torch.equal(y[keep], clean[keep])


def test_empty_sizes(device):
    w = ref.draw(device, 16, dtype=torch.float32)
    got = step(torch.empty(0, 16, device=device), w, w, torch.empty(0, 16, device=device))
    assert got["y"].shape == (0, 16) and got["dx"].shape == (0, 16) and not got["dweight"].any() and not got["dbias"].any()
    assert tritonix.layer_norm(torch.empty(4, 0, device=device)).shape == (4, 0)


def test_gradients_against_differences(device):
    rows, n, h = 6, 50, 1e-4
    parts = {"x": ref.draw(device, rows, n, dtype=torch.float32, seed=1), "weight": ref.draw(device, n, dtype=torch.float32, seed=2),
             "bias": ref.draw(device, n, dtype=torch.float32, seed=3)}
    dy = ref.draw(device, rows, n, dtype=torch.float32, seed=4)
    got = step(parts["x"], parts["weight"], parts["bias"], dy)
    want = ref.layer_norm(parts["x"], parts["weight"], parts["bias"], 1e-5, dy)
    for name, t in parts.items():
        direction = ref.draw("cpu", *t.shape, dtype=torch.float64, seed=5)
        loss = []
        for sign in (1, -1):
            p = {key: v.double().cpu() for key, v in parts.items()}
            p[name] = p[name] + sign * h * direction
            c = p["x"] - p["x"].mean(dim=1, keepdim=True)
            y = c / torch.sqrt((c * c).mean(dim=1, keepdim=True) + 1e-5) * p["weight"] + p["bias"]
            loss.append((y * dy.double().cpu()).sum())
        difference = (loss[0] - loss[1]) / (2 * h)
        bound = (want["d" + name][1] * direction.abs()).sum() + 1e-5 * want["d" + name][0].abs().sum()
        assert abs((got["d" + name].double().cpu() * direction).sum() - difference) <= bound, name


def test_only_what_is_asked_for(device):
    x, w, b, dy = (ref.draw(device, *s, dtype=torch.float32, seed=i) for i, s in enumerate(((30, 200), (200,), (200,), (30, 200))))
    want = ref.layer_norm(x, w, b, 1e-5, dy)
    for subset in (["x"], ["weight"], ["bias"], ["x", "bias"], ["weight", "bias"]):
        t = {name: v.detach().clone().requires_grad_(name in subset) for name, v in (("x", x), ("weight", w), ("bias", b))}
        y = tritonix.layer_norm(t["x"], t["weight"], t["bias"])
        for name, g in zip(subset, torch.autograd.grad(y, [t[name] for name in subset], dy)):
            ref.check(name, g, want["d" + name])
    leaf = x.detach().clone().requires_grad_(True)
    (g,) = torch.autograd.grad(tritonix.layer_norm(leaf, w, b), leaf, dy, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_from_a_graph(device):
    x, w, b, dy = (ref.draw(device, *s, seed=i) for i, s in enumerate(((300, 1000), (1000,), (1000,), (300, 1000))))
    leaves = [t.requires_grad_(True) for t in (x, w, b)]

    def once():
        y = tritonix.layer_norm(x, w, b)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = once()
    for i in range(3):
        with torch.no_grad():
            for j, t in enumerate((x, w, b, dy)):
                t.copy_(ref.draw(device, *t.shape, seed=10 * i + j))
        want = once()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(outs, want):
            assert torch.equal(a, c)
