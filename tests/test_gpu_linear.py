"""Linear layers against the definition in 64 bits: values and gradients, every activation, type and layout, sizes off every tile."""
import ctypes
import itertools

import pytest
import torch

import blocks_reference as ref
import tritonix
from tritonix_amd import _C
from tritonix_amd.ops.linear import ACTIVATIONS

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
ACTS = [None, "relu", "silu", "gelu", "gelu_tanh"]


def weight(device, k, n, dtype, layout, seed):
    w = ref.draw(device, k, n, dtype=dtype, seed=seed, scale=k ** -0.5) if layout == "nn" else \
        ref.draw(device, n, k, dtype=dtype, seed=seed, scale=k ** -0.5).t()
    return w


def step(x, w, bias, act, residual, dy):
    leaves = {"x": x, "w": w, "bias": bias, "residual": residual}
    leaves = {name: t.detach().requires_grad_(True) for name, t in leaves.items() if t is not None}
    y = tritonix.linear(leaves["x"], leaves["w"], leaves.get("bias"), activation=act, residual=leaves.get("residual"))
    grads = torch.autograd.grad(y, list(leaves.values()), dy)
    return {"y": y.detach(), **{"d" + name: g for name, g in zip(leaves, grads)}}


SIZES = [(1, 64, 64), (1, 1, 1), (2, 3, 5), (5, 8, 1), (17, 33, 65), (64, 128, 256), (33, 200, 1024), (130, 257, 96), (300, 520, 1000), (513, 770, 514),
         (257, 2, 130), (3, 1030, 2050)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("layout", ["nn", "nt"])
def test_values(device, dtype, m, n, k, layout):
    seed = m * 7 + n * 3 + k
    x, w = ref.draw(device, m, k, dtype=dtype, seed=seed), weight(device, k, n, dtype, layout, seed + 1)
    bias, residual = ref.draw(device, n, dtype=dtype, seed=seed + 2), ref.draw(device, m, n, dtype=dtype, seed=seed + 3)
    act = ACTS[seed % 5]
    for b, a, r in ((None, None, None), (bias, None, None), (None, act, None), (None, None, residual), (bias, act, residual), (bias.float(), act, None)):
        y = tritonix.linear(x, w, b, activation=a, residual=r)
        ref.check(f"y {a} bias {b is not None} residual {r is not None}", y, ref.linear(x, w, b, a, r)["y"], dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,n,k,layout", [(1, 40, 72, "nn"), (70, 96, 130, "nt"), (200, 264, 192, "nn"), (129, 65, 33, "nt"), (7, 3, 2, "nn")])
def test_gradients(device, dtype, act, m, n, k, layout):
    x, w = ref.draw(device, m, k, dtype=dtype, seed=m), weight(device, k, n, dtype, layout, 1)
    bias, residual, dy = (ref.draw(device, *s, dtype=dtype, seed=i) for i, s in ((2, (n,)), (3, (m, n)), (4, (m, n))))
    for b, r in ((bias, residual), (None, None), (bias.float(), None)):
        got = step(x, w, b, act, r, dy)
        want = ref.linear(x, w, b, act, r, dy)
        assert set(got) == set(want)
        for name in got:
            ref.check(name, got[name], want[name], b.dtype if name == "dbias" else dtype)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_gradients_against_differences(device, act):
    """Central differences of the definition in 64 bits, which knows no derivative: step h, off by h^2 / 6 of the third derivative along the direction."""
    m, n, k, h = 9, 21, 34, 1e-4
    parts = {"x": ref.draw(device, m, k, dtype=torch.float32, seed=1), "w": ref.draw(device, k, n, dtype=torch.float32, seed=2, scale=0.2),
             "bias": ref.draw(device, n, dtype=torch.float32, seed=3), "residual": ref.draw(device, m, n, dtype=torch.float32, seed=4)}
    dy = ref.draw(device, m, n, dtype=torch.float32, seed=5)
    got = step(parts["x"], parts["w"], parts["bias"], act, parts["residual"], dy)
    want = ref.linear(parts["x"], parts["w"], parts["bias"], act, parts["residual"], dy)
    for name, t in parts.items():
        direction = ref.draw("cpu", *t.shape, dtype=torch.float64, seed=6)
        loss = []
        for sign in (1, -1):
            p = {key: v.double().cpu() for key, v in parts.items()}
            p[name] = p[name] + sign * h * direction
            z = p["x"] @ p["w"] + p["bias"]
            loss.append(((ref.activation(z, act) + p["residual"]) * dy.double().cpu()).sum())
        difference = (loss[0] - loss[1]) / (2 * h)
        mine = (got["d" + name].double().cpu() * direction).sum()
        bound = (want["d" + name][1] * direction.abs()).sum() + 1e-5 * want["d" + name][0].abs().sum()
        assert abs(mine - difference) <= bound, (name, float(mine), float(difference), float(bound))


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignments(device, dtype):
    m, n, k = 77, 90, 130
    big = ref.draw(device, 200, 400, dtype=dtype, seed=1)
    w0, b0, r0 = ref.draw(device, 300, 200, dtype=dtype, seed=2, scale=0.1), ref.draw(device, 200, dtype=dtype, seed=3), ref.draw(device, 100, 200, dtype=dtype, seed=4)
    xs = {"pitch": big[:m, 3:3 + k], "every other row": big[:2 * m:2, :k], "column-major": big[:k, :m].t(), "every other column": big[:m, :2 * k:2],
          "one row for all": big[:1, :k].expand(m, k), "reversed": big[:m, :k].flip(0)}
    ws = {"pitch": w0[5:5 + k, 1:1 + n], "transposed": w0[:n, :k].t(), "every other column": w0[:k, :2 * n:2], "one column for all": w0[:k, :1].expand(k, n)}
    for (nx, x), (nw, w) in itertools.product(xs.items(), ws.items()):
        bias, residual = b0[:2 * n:2], r0[:m, 7:7 + n]
        got = step(x, w, bias, "silu", residual, r0[:m, 50:50 + n])
        want = ref.linear(x, w, bias, "silu", residual, r0[:m, 50:50 + n])
        for name in got:
            ref.check(f"{nx}, {nw}: {name}", got[name], want[name], dtype)


def test_leading_dimensions(device):
    x, w, b = ref.draw(device, 2, 5, 3, 48, seed=1), ref.draw(device, 48, 24, seed=2, scale=0.2), ref.draw(device, 24, seed=3)
    r = ref.draw(device, 2, 5, 3, 24, seed=4)
    y = tritonix.linear(x, w, b, "gelu", r)
    assert y.shape == (2, 5, 3, 24)
    assert torch.equal(y.reshape(30, 24), tritonix.linear(x.reshape(30, 48), w, b, "gelu", r.reshape(30, 24)))
    one = tritonix.linear(x[0, 0, 0], w, b)
    assert one.shape == (24,)
    ref.check("vector", one[None], ref.linear(x[0, 0, :1], w, b)["y"])
    xg = x.clone().requires_grad_(True)
    tritonix.linear(xg, w, b, "gelu", r).sum().backward()
    assert xg.grad.shape == x.shape


@pytest.mark.parametrize("dtype", DTYPES)
def test_empty_sizes(device, dtype):
    w, b = ref.draw(device, 16, 8, dtype=dtype, seed=1), ref.draw(device, 8, dtype=dtype, seed=2)
    assert tritonix.linear(torch.empty(0, 16, dtype=dtype, device=device), w, b, "silu").shape == (0, 8)
    assert tritonix.linear(ref.draw(device, 3, 16, dtype=dtype), w[:, :0], b[:0]).shape == (3, 0)
    # no k: the bias alone goes through the activation
    x0, r = torch.empty(3, 0, dtype=dtype, device=device), ref.draw(device, 3, 8, dtype=dtype, seed=3)
    got = step(x0, w[:0], b, "gelu", r, r)
    want = ref.linear(x0, w[:0], b, "gelu", r, r)
    for name in got:
        ref.check(name, got[name], want[name])
    assert torch.equal(tritonix.linear(x0, w[:0]), torch.zeros(3, 8, dtype=dtype, device=device))
    # no rows: the gradients of weight and bias are zeros
    got = step(torch.empty(0, 16, dtype=dtype, device=device), w, b, "relu", None, torch.empty(0, 8, dtype=dtype, device=device))
    assert got["dx"].shape == (0, 16) and not got["dw"].any() and not got["dbias"].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_numbers_that_are_none(device, dtype):
    """An infinity or a NaN in a row of x, of the residual or in the bias shows in the outputs it enters and in no others."""
    m, n, k = 70, 130, 96
    x, w, b, r = (ref.draw(device, *s, dtype=dtype, seed=i) for i, s in enumerate(((m, k), (k, n), (n,), (m, n))))
    clean = tritonix.linear(x, w, b, "relu", r)
    x[3, 5], r[20, 7], b[9] = float("nan"), float("inf"), float("nan")
    y = tritonix.linear(x, w, b, "relu", r)
    touched = torch.zeros(m, n, dtype=torch.bool, device=device)
    touched[3], touched[20, 7], touched[:, 9] = True, True, True
    assert torch.equal(y[~touched], clean[~touched])
    assert y[3].isnan().all() and y[:, 9].isnan().all() and torch.isposinf(y[20, 7])
    z = torch.tensor([[-3e4, 3e4, 0.0, -0.0]], dtype=dtype, device=device)
    eye = torch.eye(4, dtype=dtype, device=device)
    for act in ACTS[1:]:
        g = step(z, eye, None, act, None, torch.ones_like(z))
        assert torch.equal(g["y"], torch.tensor([[0.0, 3e4, 0.0, 0.0]], dtype=dtype, device=device)), act
        assert torch.equal(g["dx"][0, :2], torch.tensor([0.0, 1.0], dtype=dtype, device=device)), act


def args_of(x, w, bias=None, act=None):
    a = _C.LinearArgs()
    a.x, a.w, a.bias = x.data_ptr(), w.data_ptr(), bias.data_ptr() if bias is not None else None
    a.m, a.k = x.shape
    a.n = w.shape[1]
    a.stride_xm, a.stride_xk, a.stride_wk, a.stride_wn = *x.stride(), *w.stride()
    a.dtype = {torch.float16: _C.F16, torch.bfloat16: _C.BF16, torch.float32: _C.F32}[x.dtype]
    a.bias_dtype, a.activation = a.dtype, ACTIVATIONS[act]
    return a


# sizes that the built-in choice gives each of its tiles, cut along k and not
ROUTED = [(8, 512, 512), (24, 4096, 4096), (48, 512, 4096), (64, 8192, 512), (100, 1000, 600), (256, 384, 5000), (500, 3000, 256), (1024, 1024, 1024),
          (1500, 2000, 328), (2048, 2048, 256), (4096, 4096, 64), (768, 5000, 192), (5000, 700, 200)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", ROUTED)
@pytest.mark.parametrize("layout", ["nn", "nt"])
def test_tiles_of_the_built_in_choice(device, dtype, m, n, k, layout):
    x, w = ref.draw(device, m, k, dtype=dtype, seed=1), weight(device, k, n, dtype, layout, 2)
    bias, residual = ref.draw(device, n, dtype=dtype, seed=3), ref.draw(device, m, n, dtype=dtype, seed=4)
    info = (ctypes.c_int32 * 5)()
    route = _C.load().tnx_linear_route(ctypes.byref(args_of(x, w, bias, "silu")), info)
    if m > 16:
        assert route == _C.LINEAR_ROUTE_FUSED, (route, list(info))
    for _ in range(2):                     # (a second call finds the counters of a cut as the first left them)
        y = tritonix.linear(x, w, bias, "silu", residual)
    # a sample of rows: the definition of all of them would take the CPU minutes
    rows = torch.unique(torch.cat([torch.arange(0, m, max(1, m // 37)), torch.tensor([m - 1])]))
    at = rows.to(device)
    ref.check(f"tile {list(info)}", y[at], ref.linear(x[at], w, bias, "silu", residual[at])["y"], dtype)


def strided(device, rows, cols, dtype, seed, pitch, offset, scale=1.0):
    """Rows of cols elements, pitch apart, the first offset elements into its storage; NaN between and around them."""
    whole = torch.full((offset + rows * pitch + 8,), float("nan"), dtype=dtype, device=device)
    out = whole[offset:offset + rows * pitch].view(rows, pitch)[:, :cols]
    out.copy_(ref.draw(device, rows, cols, dtype=dtype, seed=seed, scale=scale))
    return out


FEW = [(1, 1, 1), (1, 8, 1), (2, 64, 64), (1, 8, 4097), (7, 1024, 4099), (5, 130, 4600), (2, 8200, 77), (4, 9001, 1030), (8, 500, 4608), (1, 72, 4100), (8, 520, 2500), (6, 1001, 5000), (3, 9000, 1025), (1, 5, 7), (3, 9, 63), (4, 100, 257), (4, 4095, 520), (1, 4097, 136), (4, 4100, 1100), (5, 4104, 640), (8, 4099, 1026), (8, 33, 8192), (5, 17, 31), (8, 300, 2050),
       (9, 50, 64), (16, 129, 1025), (13, 4500, 513), (16, 16, 4608), (1, 70, 9000)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", FEW)
@pytest.mark.parametrize("pad,offset", [(0, 0), (64, 64), (1, 3), (8, 8)])
@pytest.mark.parametrize("layout", ["nt", "nn"])
def test_few_rows(device, dtype, m, n, k, pad, offset, layout):
    """Blocks and steps that end inside the matrix, rows of the weight on lines of memory and off them; what lies between rows is never used."""
    x = strided(device, m, k, dtype, 1, k + pad, offset)
    rows, cols = (n, k) if layout == "nt" else (k, n)
    w = strided(device, rows, cols, dtype, 2, (cols + 63) // 64 * 64 if pad == 64 else cols + pad, offset, k ** -0.5)
    w = w.t() if layout == "nt" else w
    bias, residual = ref.draw(device, n, dtype=dtype, seed=3), ref.draw(device, m, n, dtype=dtype, seed=4)
    args = args_of(x, w, bias, "gelu")
    route = _C.load().tnx_linear_route(ctypes.byref(args), None)
    if layout == "nt" and (m == 1 or m <= 4 and k <= 8192) and (dtype == torch.float32 or n * k <= 1 << 20):
        assert route == _C.LINEAR_ROUTE_STREAM
    elif layout == "nn" and m <= 8 and 8 <= n <= 1024 and k >= 4096 and dtype != torch.float32 or layout == "nn" and m <= 4 and n > 8192 and k <= 4096 and dtype == torch.float32:
        assert route == _C.LINEAR_ROUTE_STREAM_ROWS
    ref.check("y", tritonix.linear(x, w, bias, "gelu", residual), ref.linear(x, w, bias, "gelu", residual)["y"], dtype)
    plain = tritonix.linear(x, w)
    ref.check("product", plain, ref.linear(x, w)["y"], dtype)
    # a row's numbers are its own: one that is not a number stays in its row, and in its column of the weight
    x[m // 2, k - 1] = float("inf")
    y = tritonix.linear(x, w)
    others = torch.arange(m, device=device) != m // 2
    assert torch.equal(y[others], plain[others]) and not y[m // 2].isfinite().any()
    x[m // 2, k - 1] = 1.0
    w[0, n - 1] = float("nan")
    y = tritonix.linear(x, w)
    assert torch.equal(y[others, :n - 1], plain[others, :n - 1]) and y[:, n - 1].isnan().all()


@pytest.mark.parametrize("m", [40, 3])
def test_same_bits_every_time_and_from_a_graph(device, m):
    """Values and gradients from a captured graph, replayed with the program's own work between, are the eager ones bit for bit."""
    n, k = 1000, 2304                                # K is cut: counters in the graph's own workspace
    x, w, b, r, dy = (ref.draw(device, *s, seed=i, scale=0.1) for i, s in enumerate(((m, k), (k, n), (n,), (m, n), (m, n))))
    leaves = [t.requires_grad_(True) for t in (x, w, b, r)]

    def once():
        y = tritonix.linear(x, w, b, "gelu", r)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    for _ in range(2):                                      # two graphs of one stream
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            graphs.append((graph, once()))
    for i in range(3):
        with torch.no_grad():
            for j, t in enumerate((x, w, b, r, dy)):
                t.copy_(ref.draw(device, *t.shape, seed=10 * i + j, scale=0.1))
        want = once()
        torch.cuda.synchronize()
        for s, (graph, _) in zip((torch.cuda.Stream(), torch.cuda.Stream()), graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for _, outs in graphs:
            for a, c in zip(outs, want):
                assert torch.equal(a, c)


def test_products_of_a_graph_share_their_counters(device):
    """Several products that are cut along k in one graph, some on a second stream of it, eager ones and another graph of the same stream between:
    every replay gives the eager bits."""
    sizes = [(40, 1000, 2304), (24, 4096, 4096), (3, 512, 8192), (64, 700, 5000)]
    w = [ref.draw(device, k, n, seed=i, scale=k ** -0.5) for i, (m, n, k) in enumerate(sizes)]
    x = [ref.draw(device, m, k, seed=10 + i) for i, (m, n, k) in enumerate(sizes)]

    def products(which):
        return [tritonix.linear(x[i], w[i], activation="silu") for i in which]

    side, second = torch.cuda.Stream(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        products(range(4))
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = products((0, 1))
            second.wait_stream(side)
            with torch.cuda.stream(second):
                outs += products((2, 3, 2))
            outs += products((3, 2))
            side.wait_stream(second)
            outs += products((1, 0))
        graphs.append((graph, outs))
        with torch.cuda.stream(side):
            products(range(4))
        torch.cuda.synchronize()
    for turn in range(4):
        for i, t in enumerate(x):
            t.copy_(ref.draw(device, *t.shape, seed=100 * turn + i))
        want = [products((i,))[0] for i in (0, 1, 2, 3, 2, 3, 2, 1, 0)]
        for graph, outs in graphs:
            graph.replay()
            products((turn % 4,))
            torch.cuda.synchronize()
            for a, c in zip(outs, want):
                assert torch.equal(a, c)


def test_on_another_stream(device):
    x, w, b = (ref.draw(device, *s, seed=i) for i, s in enumerate(((33, 2048), (2048, 512), (512,))))
    want = tritonix.linear(x, w, b, "silu")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = tritonix.linear(x, w, b, "silu")
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


def test_only_what_is_asked_for(device):
    """Gradients of any subset of the inputs; the same tensor as residual and input; no second derivative."""
    m, n, k = 20, 32, 32
    x, w, b, r, dy = (ref.draw(device, *s, dtype=torch.float32, seed=i) for i, s in enumerate(((m, k), (k, n), (n,), (m, n), (m, n))))
    want = ref.linear(x, w, b, "gelu", r, dy)
    names = ["x", "w", "bias", "residual"]
    for count in range(1, 5):
        for subset in itertools.combinations(names, count):
            t = {name: v.detach().clone().requires_grad_(name in subset) for name, v in zip(names, (x, w, b, r))}
            y = tritonix.linear(t["x"], t["w"], t["bias"], "gelu", t["residual"])
            for name, g in zip(subset, torch.autograd.grad(y, [t[name] for name in subset], dy)):
                ref.check(name, g, want["d" + name])
    both = x.detach().clone().requires_grad_(True)
    (g,) = torch.autograd.grad(tritonix.linear(both, w, b, "gelu", both), both, dy)
    w2 = ref.linear(x, w, b, "gelu", x, dy)
    ref.check("x and residual", g, (w2["dx"][0] + w2["dresidual"][0], w2["dx"][1] + 2.0 ** -24 * (w2["dx"][0] + w2["dresidual"][0]).abs() + 1e-6))
    y = tritonix.linear(both, w, b, "gelu")
    (g,) = torch.autograd.grad(y, both, dy, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_the_residuals_gradient_is_its_own(device):
    """A gradient that is handed on as it is, accumulated into twice, leaves the caller's tensor alone."""
    x, w, r = (ref.draw(device, *s, dtype=torch.float32, seed=i).requires_grad_(True) for i, s in enumerate(((4, 16), (16, 32), (4, 32))))
    dy = ref.draw(device, 4, 32, dtype=torch.float32, seed=5)
    kept = dy.clone()
    for _ in range(2):
        tritonix.linear(x, w, None, "silu", r).backward(dy)
    assert torch.equal(r.grad, kept + kept) and torch.equal(dy, kept)
    assert r.grad.data_ptr() != dy.data_ptr()


def test_the_interpreters_path_gives_the_same(device, monkeypatch):
    """Calls that csrc/launch.cpp does not take: the same kernels, the same bits."""
    from tritonix_amd.ops import mx, native

    x, w, b, r, dy = (ref.draw(device, *s, seed=i) for i, s in enumerate(((40, 64), (64, 2304), (2304,), (40, 2304), (40, 2304))))
    bounds, e = torch.tensor([0, 7, 7, 40], dtype=torch.int32, device=device), ref.draw(device, 3, 64, 48, seed=9)

    def everything():
        out = step(x, w, b, "gelu", r, dy)
        leaves = [t.detach().requires_grad_(True) for t in (x, e)]
        y = tritonix.grouped_matmul(*leaves, bounds)
        more = [y.detach(), *torch.autograd.grad(y, leaves, dy[:, :48])]
        leaves = [t.detach().requires_grad_(True) for t in (r, b, b)]
        y = tritonix.layer_norm(*leaves)
        return [*out.values(), *more, y.detach(), *torch.autograd.grad(y, leaves, dy), tritonix.linear(x, w, b), tritonix.layer_norm(x), tritonix.grouped_matmul(x, e, bounds)]

    first = everything()
    assert native.module is not mx._Interpreter, "the native side is not in use"
    monkeypatch.setattr(native, "module", mx._Interpreter)
    for a, c in zip(first, everything()):
        assert torch.equal(a, c)
