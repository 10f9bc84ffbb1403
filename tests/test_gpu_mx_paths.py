"""The two host paths of the microscaled and routing calls, the native one and the interpreter's, are one operator: the same bits, the same refusals."""
import ctypes

import pytest
import torch

import tritonix
from tritonix_amd import _C
from tritonix_amd.ops import mx

pytestmark = pytest.mark.gpu


class Counting:
    """The native module, with what it answered (True) and handed back (False) noted per function."""

    def __init__(self, module):
        self.module, self.answers = module, []

    def __getattr__(self, name):
        def call(*args):
            out = getattr(self.module, name)(*args)
            self.answers.append((name, out is not None))
            return out
        return call


def both(monkeypatch, call, asked):
    """``call`` natively, which answers the functions named in ``asked``, and through the interpreter."""
    counting = Counting(mx.find_native())
    monkeypatch.setattr(mx, "native", counting)
    got = call()
    assert [name for name, answered in counting.answers if answered] == asked, counting.answers
    monkeypatch.setattr(mx, "native", mx._Interpreter)
    want = call()
    assert len(got) == len(want)
    for g, w in zip(got, want):
        assert g.dtype == w.dtype and g.shape == w.shape and torch.equal(g, w)


def rand(device, *shape, dtype=torch.bfloat16, seed=0):
    return torch.randn(shape, generator=torch.Generator("cpu").manual_seed(seed)).to(dtype).to(device)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("dim", [0, 1])
def test_quantisation(device, monkeypatch, dtype, dim):
    x = rand(device, 70, 300, dtype=dtype)

    def call():
        t = tritonix.mx_quantize(x, dim=dim)
        return t.codes, tritonix.mx_dequantize(t, dtype)
    both(monkeypatch, call, ["mx_quantize", "mx_dequantize"])


@pytest.mark.parametrize("m", [1, 2, 3, 40, 200])
@pytest.mark.parametrize("wide", [False, True])
def test_products(device, monkeypatch, m, wide):
    x = rand(device, m, 600)[:, :300] if wide else rand(device, m, 300)
    w = mx.mx_quantize(rand(device, 300, 132, seed=1), dim=0)
    both(monkeypatch, lambda: (tritonix.mx_matmul(x, w), tritonix.mx_glu(x, w), tritonix.mx_glu(x, w, "none")), ["mx_product"] * 3)


@pytest.mark.parametrize("size", [(40, 500, 14336), (100, 1100, 14336), (130, 2050, 9000), (200, 1030, 17000)], ids=str)
@pytest.mark.parametrize("epilogue", ["plain", "silu"])
def test_products_with_k_in_parts(device, monkeypatch, size, epilogue):
    """The same sums, added up in another order: against the product without the scratch, and the native path against the interpreter's."""
    m, n, k = size
    a, w = mx.mx_quantize(rand(device, m, k)), mx.mx_quantize(rand(device, k, n, seed=1), dim=0)
    call = (lambda x: tritonix.mx_matmul(x, w, out_dtype=torch.float32)) if epilogue == "plain" else (lambda x: tritonix.mx_glu(x, w, out_dtype=torch.float32))
    lib = _C.load()
    got = call(a)
    out = torch.empty_like(got)
    g = mx.gemm_args(a, w, out, _C.EPI_NONE if epilogue == "plain" else _C.EPI_GLU_SILU)
    g.stream = torch.cuda.current_stream().cuda_stream
    assert lib.tnx_mx_gemm_workspace_bytes(ctypes.byref(g)) > 0
    assert lib.tnx_mx_gemm(ctypes.byref(g)) == _C.OK            # without scratch
    product = tritonix.mx_matmul(a, w, out_dtype=torch.float32)
    # sums of k terms of magnitude up to the largest entry's scale, rounded in two orders of 2^-24 each; the gate's slope is at most 1.1
    scale = (tritonix.mx_dequantize(a, torch.float32).abs() @ tritonix.mx_dequantize(w, torch.float32).abs()).max()
    bound = float(scale) * (k // 64 + 16) * 2.0 ** -23
    bound = bound if epilogue == "plain" else 2.2 * bound * float(product.abs().max())
    assert float((got - out).abs().max()) <= bound
    if epilogue == "plain":
        x = rand(device, m, k)
        both(monkeypatch, lambda: (tritonix.mx_matmul(x, w),), ["mx_product"])


def test_linear(device, monkeypatch):
    x, w, dy = rand(device, 65, 130).requires_grad_(True), rand(device, 130, 66, seed=1).requires_grad_(True), rand(device, 65, 66, seed=2)

    def call():
        y = tritonix.mx_linear(x, w)
        return (y.detach(), *torch.autograd.grad(y, (x, w), dy))
    counting = Counting(mx.find_native())
    monkeypatch.setattr(mx, "native", counting)
    got = call()
    assert counting.answers == [("mx_linear", True)]
    monkeypatch.setattr(mx, "native", mx._Interpreter)
    assert all(torch.equal(g, h) for g, h in zip(got, call()))


def test_linear_of_one_operand_that_is_trained(device):
    x, w, dy = rand(device, 65, 130), rand(device, 130, 66, seed=1), rand(device, 65, 66, seed=2)
    xg, wg = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dx, dw = torch.autograd.grad(tritonix.mx_linear(xg, wg), (xg, wg), dy)
    assert torch.equal(torch.autograd.grad(tritonix.mx_linear(xg, w), xg, dy)[0], dx)
    assert torch.equal(torch.autograd.grad(tritonix.mx_linear(x, wg), wg, dy)[0], dw)
    # a gradient that is one number, broadcast with strides of zero
    (one,) = torch.autograd.grad(tritonix.mx_linear(xg, w).sum(), xg)
    assert torch.equal(one, torch.autograd.grad(tritonix.mx_linear(xg, w), xg, torch.ones_like(dy))[0])


@pytest.mark.parametrize("tokens", [1, 9, 300])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_routing(device, monkeypatch, tokens, dtype):
    logits, bias, grad = rand(device, tokens, 48, dtype=dtype), rand(device, 48, dtype=torch.float32, seed=1), rand(device, tokens, 4, dtype=torch.float32)

    def call():
        r = tritonix.moe_route(logits, 4)
        s = tritonix.moe_route(logits, 4, scoring="sigmoid", bias=bias, num_groups=4, top_groups=2, group_top=2, scale=2.5)
        return r.weights, r.experts, r.offsets, r.rows, s.weights, s.experts, s.offsets, s.order, s.rows, tritonix.moe_route_backward(grad, logits, s)
    both(monkeypatch, call, ["moe_route", "moe_route", "moe_backward"])


@pytest.mark.parametrize("tokens", [1, 2, 30, 200])
def test_block(device, monkeypatch, tokens):
    x = rand(device, tokens, 128)
    w12, w3 = (tritonix.mx_quantize(rand(device, *s, seed=1), dim=-2) for s in ((6, 128, 192), (6, 96, 128)))
    r = tritonix.moe_route(rand(device, tokens, 6, dtype=torch.float32, seed=2), 2)
    both(monkeypatch, lambda: (tritonix.moe_glu(x, w12, r), tritonix.moe_ffn(x, w12, w3, r)), ["mx_product"] * 3)


def test_a_changed_routing_is_refused(device):
    x = rand(device, 5, 64)
    w12, w3 = (tritonix.mx_quantize(rand(device, *s), dim=-2) for s in ((3, 64, 64), (3, 32, 64)))
    made = tritonix.moe_route(rand(device, 5, 3, dtype=torch.float32), 2)
    h = tritonix.moe_glu(x, w12, made)
    up, down = (lambda r: tritonix.moe_glu(x, w12, r)), (lambda r: tritonix.moe_down(h, w3, r))         # each with the fields that it reads
    for call, field, value in ((down, "weights", made.weights.half()), (down, "weights", made.weights[:, :1]), (down, "weights", made.weights.cpu()),
                               (down, "rows", made.rows.t().contiguous().t()), (down, "offsets", made.offsets[:3]), (up, "offsets", made.offsets[:3]),
                               (up, "order", made.order.long()), (up, "order", made.order.cpu())):
        with pytest.raises(ValueError):
            call(tritonix.Routing(**{**vars(made), field: value}))
    with pytest.raises(ValueError):
        tritonix.moe_route_backward(made.weights, rand(device, 5, 3), tritonix.Routing(**{**vars(made), "experts": made.experts.long()}))


def test_offsets_and_rows_out_of_range_stay_inside(device):
    """A plan that was overwritten gives wrong sums, not reads outside: rows past the end are nobody's, sources clamp."""
    x = rand(device, 5, 64)
    w12, w3 = (tritonix.mx_quantize(rand(device, *s), dim=-2) for s in ((3, 64, 64), (3, 32, 64)))
    made = tritonix.moe_route(rand(device, 5, 3, dtype=torch.float32), 2)
    r = tritonix.Routing(**{**vars(made), "offsets": torch.tensor([0, 7, 3, 1 << 30], dtype=torch.int32, device=device),
                            "order": torch.full_like(made.order, 1 << 30), "rows": torch.full_like(made.rows, 1 << 30)})
    assert tritonix.moe_glu(x, w12, r).shape == (10, 32)
    out = tritonix.moe_down(rand(device, 10, 32), w3, r)
    torch.cuda.synchronize()
    assert (out == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("shape", [(1, 40), (40, 1), (2, 2), (33, 31), (64, 256), (255, 257), (300, 129), (513, 700), (31, 1030)], ids=str)
@pytest.mark.parametrize("order", ["rows", "columns", "neither"])
def test_both_quantisations_at_once_are_the_two(device, dtype, shape, order):
    m, k = shape
    x = rand(device, m, k, dtype=dtype)
    x[0, :min(k, 32)] = 0
    x[m // 2, k // 2] = float("inf")
    x[m - 1, k - 1] = float("nan")
    if order == "columns":
        x = x.t().contiguous().t()
    elif order == "neither":
        x = x.repeat_interleave(2, 0).repeat_interleave(2, 1)[::2, ::2]
    along, across = tritonix.mx_quantize(x, dim=-1), tritonix.mx_quantize(x, dim=-2)
    got, other = mx.MXTensor.empty(None, m, k, -1, device), mx.MXTensor.empty(None, k, m, -2, device)
    for t in (got, other):
        t.buffer.fill_(0xA5)
    a = mx._mx_args(x, got, mx.dtype_code("test", dtype))
    a.stream = torch.cuda.current_stream().cuda_stream
    assert _C.load().tnx_mx_quantize_both(ctypes.byref(a), other.codes_ptr, other.scales_ptr) == _C.OK
    for g, w in ((got, along), (other, across)):
        assert torch.equal(g.codes, w.codes)
        assert torch.equal(tritonix.mx_dequantize(g, torch.float32).nan_to_num(123.0), tritonix.mx_dequantize(w, torch.float32).nan_to_num(123.0))
        # scales of every row and slab, the padding's among them (rows past the last and a slab past an odd count belong to nobody)
        slabs = -(-g.k // 256)
        view = lambda t: t.scales.view(-1, -(-slabs // 2), 32, 2, 8).permute(0, 2, 1, 3, 4).reshape(-1, -(-slabs // 2) * 2, 8)[:g.rows, :slabs]      # noqa: E731
        assert torch.equal(view(g), view(w))


def test_linear_keeps_what_it_was_called_with(device):
    """The operands may change between the passes: the gradients are those of the values the product saw."""
    x, w, dy = rand(device, 65, 130).requires_grad_(True), rand(device, 130, 66, seed=1).requires_grad_(True), rand(device, 65, 66, seed=2)
    want = torch.autograd.grad(tritonix.mx_linear(x, w), (x, w), dy)
    y = tritonix.mx_linear(x, w)
    with torch.no_grad():
        w.zero_()
    first = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    again = torch.autograd.grad(y, (x, w), dy)
    for g, h, i in zip(want, first, again):
        assert torch.equal(g, h) and torch.equal(g, i)
    with torch.no_grad():
        assert not tritonix.mx_linear(x, w).requires_grad


def test_linear_steps_in_threads_and_streams(device):
    """Backward passes of two graphs on a stream of their own each."""
    x, w, dy = rand(device, 300, 260), rand(device, 260, 520, seed=1), rand(device, 300, 520, seed=2)
    xs = x.clone().requires_grad_(True)
    want = torch.autograd.grad(tritonix.mx_linear(xs, w), xs, dy)[0]
    torch.cuda.synchronize()
    got = []
    for _ in range(2):
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            got.append(torch.autograd.grad(tritonix.mx_linear(xs, w), xs, dy)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_the_example_runs(device, capsys):
    import os
    import runpy

    main = runpy.run_path(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "routed_ffn.py"))["main"]
    worst, largest = main(tokens=300, width=256, inner=128, experts=8, top_k=2, device=device)
    assert 0 < largest < float("inf") and 0 <= worst < float("inf")
    assert "rows per expert" in capsys.readouterr().out


@pytest.mark.parametrize("native", [True, False])
def test_second_derivatives_are_an_error(device, monkeypatch, native):
    """Not a silent zero: the gradients are computed, and differentiating them says so."""
    if not native:
        monkeypatch.setattr(mx, "native", mx._Interpreter)
    x, w = rand(device, 33, 64, dtype=torch.float32).requires_grad_(True), rand(device, 64, 40, dtype=torch.float32, seed=1).requires_grad_(True)
    want = torch.autograd.grad(tritonix.mx_linear(x, w).square().sum(), (x, w))
    got = torch.autograd.grad(tritonix.mx_linear(x, w).square().sum(), (x, w), create_graph=True)
    assert all(torch.equal(g, h) for g, h in zip(got, want))
    with pytest.raises(RuntimeError):
        got[0].sum().backward()
    (one,) = torch.autograd.grad(tritonix.mx_linear(x, w.detach()).square().sum(), x, create_graph=True)
    assert torch.equal(one, want[0])
    with pytest.raises(RuntimeError):
        one.sum().backward()
    logits = rand(device, 9, 16, dtype=torch.float32).requires_grad_(True)
    (g,) = torch.autograd.grad(tritonix.moe_route(logits, 3).weights.square().sum(), logits, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.parametrize("tokens,dtype", [(1, torch.float32), (40, torch.bfloat16), (2000, torch.float32)], ids=str)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_routing_in_the_graph(device, monkeypatch, tokens, dtype, scoring):
    logits = rand(device, tokens, 48, dtype=dtype).requires_grad_(True)
    bias, grad = rand(device, 48, dtype=torch.float32, seed=1), rand(device, tokens, 4, dtype=torch.float32, seed=2)

    def call():
        r = tritonix.moe_route(logits, 4, scoring=scoring, bias=bias, renormalize=False, scale=2.0)
        assert r.weights.requires_grad and not any(t.requires_grad for t in (r.experts, r.offsets, r.order, r.rows))
        (g,) = torch.autograd.grad(r.weights, logits, grad.t().contiguous().t(), retain_graph=True)
        (h,) = torch.autograd.grad(r.weights.sum(), logits)              # (strides of zero)
        return r.weights.detach(), r.experts, r.offsets, r.order, r.rows, g, h
    both(monkeypatch, call, ["moe_route"])
    r = tritonix.moe_route(logits, 4, scoring=scoring, bias=bias, renormalize=False, scale=2.0)
    explicit = tritonix.moe_route_backward(grad, logits.detach(), r)
    assert torch.equal(torch.autograd.grad(r.weights, logits, grad)[0], explicit)
