"""Linear layers, normalisation and grouped products in the autograd graph, natively and through the interpreter: which operands are kept, and which calls have no derivative."""
import itertools

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import blocks_reference as ref
import tritonix
from tritonix_amd.ops import mx, native

pytestmark = pytest.mark.gpu
F32 = torch.float32


@pytest.fixture(params=["native", "interpreter"])
def side(request, monkeypatch, device):
    tritonix.layer_norm(torch.zeros(2, 16, device=device))            # (finds the native side)
    assert native.module is not mx._Interpreter, "the native side is not in use"
    if request.param == "interpreter":
        monkeypatch.setattr(native, "module", mx._Interpreter)
    return request.param


# what a gradient of each of the inputs reads of the others (and of itself)
READS = {"linear": {"x": {"w"}, "w": {"x"}, "bias": set(), "residual": set()}, "norm": {"x": {"x", "weight"}, "weight": {"x"}, "bias": set()}, "grouped": {"x": {"w", "offsets"}, "w": {"x", "offsets"}}}


def inputs(device, op):
    d = lambda i, *s, scale=1.0: ref.draw(device, *s, dtype=F32, seed=i, scale=scale)  # noqa: E731
    if op == "linear":
        return {"x": d(1, 40, 48), "w": d(2, 48, 64, scale=0.1), "bias": d(3, 64), "residual": d(4, 40, 64)}, d(5, 40, 64)
    if op == "norm":
        return {"x": d(1, 40, 300), "weight": d(2, 300), "bias": d(3, 300)}, d(4, 40, 300)
    return {"x": d(1, 40, 48), "w": d(2, 3, 48, 64, scale=0.1), "offsets": torch.tensor([1, 20, 20, 38], dtype=torch.int32, device=device)}, d(3, 40, 64)


def call(op, t, act):
    if op == "linear":
        return tritonix.linear(t["x"], t["w"], t["bias"], act, t["residual"])
    return tritonix.layer_norm(t["x"], t["weight"], t["bias"]) if op == "norm" else tritonix.grouped_matmul(t["x"], t["w"], t["offsets"])


def definition(op, t, dy, act):
    if op == "linear":
        return ref.linear(t["x"], t["w"], t["bias"], act, t["residual"], dy)
    return ref.layer_norm(t["x"], t["weight"], t["bias"], 1e-5, dy) if op == "norm" else ref.grouped(t["x"], t["w"], t["offsets"], dy)


@pytest.mark.parametrize("op,act", [("linear", None), ("linear", "gelu"), ("norm", None), ("grouped", None)])
def test_operands_that_no_gradient_reads_may_change(device, side, op, act):
    """Before the backward pass each operand that the gradients asked for do not read is changed in place: they are what they were.  One that they read
    is missed."""
    given, dy = inputs(device, op)
    names = [name for name in given if name != "offsets"]
    want = definition(op, given, dy, act)
    for asked in itertools.chain.from_iterable(itertools.combinations(names, c) for c in range(1, len(names) + 1)):
        read = set().union(*(READS[op][name] for name in asked))
        for changed in given:
            t = {name: v.detach().clone() for name, v in given.items()}
            leaves = [t[name].requires_grad_(True) for name in asked]
            y = call(op, t, act)
            with torch.no_grad():
                t[changed].mul_(3)
            if changed in read:
                with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                    torch.autograd.grad(y, leaves, dy)
                continue
            for name, g in zip(asked, torch.autograd.grad(y, leaves, dy)):
                ref.check(f"{asked}, {changed} changed: d{name}", g, want["d" + name])


@pytest.mark.parametrize("layout", ["nn", "nt"])
@pytest.mark.parametrize("op", ["linear", "grouped"])
def test_a_weights_gradient_has_its_layout(device, side, op, layout):
    """Also where x asks for no gradient, and the weight is not kept for one."""
    given, dy = inputs(device, op)
    last = given["w"] if layout == "nn" else given["w"].transpose(-1, -2).contiguous().transpose(-1, -2)
    for x_too in (False, True):
        t = {**given, "x": given["x"].detach().requires_grad_(x_too), "w": last.detach().requires_grad_(True)}
        (dw,) = torch.autograd.grad(call(op, t, None), (t["w"],), dy)
        ref.check("dw", dw, definition(op, given, dy, None)["dw"])
        assert dw.stride() == last.stride()


@pytest.mark.parametrize("op", ["linear", "norm", "grouped"])
def test_forward_mode_is_refused(device, side, op):
    """A tangent is refused, with gradients asked for and without, on any of the floating operands and on the gradient that comes back."""
    given, dy = inputs(device, op)
    names = [name for name in given if name != "offsets"]
    clean = call(op, given, "silu")
    with forward_ad.dual_level():
        for name in names:
            for leaf in (False, True):
                t = {k: v.detach().clone().requires_grad_(leaf and k != "offsets") for k, v in given.items()}
                t[name] = forward_ad.make_dual(t[name], torch.ones_like(t[name]))
                with pytest.raises(RuntimeError, match="forward"):
                    call(op, t, "silu")
                with torch.no_grad(), pytest.raises(RuntimeError, match="forward"):
                    call(op, t, "silu")
        t = {k: v.detach().clone() for k, v in given.items()}
        t["x"].requires_grad_(True)
        y = call(op, t, "silu")
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y, t["x"], forward_ad.make_dual(dy, torch.ones_like(dy)))
        # an operand without a tangent is as ever
        assert torch.equal(call(op, given, "silu"), clean)
    assert torch.equal(call(op, given, "silu"), clean)


@pytest.mark.parametrize("op", ["linear", "norm", "grouped"])
def test_negated_views(device, side, op):
    """A tensor that torch holds as the negative of its memory (the imaginary part of a conjugate) counts with its sign."""
    given, dy = inputs(device, op)
    names = [name for name in given if name != "offsets"]
    for name in names:
        negated = torch._neg_view(given[name])
        assert negated.is_neg()
        t = {**given, name: -given[name]}
        want = call(op, t, "silu")
        assert torch.equal(call(op, {**given, name: negated}, "silu"), want)
        leaf = given[name].detach().clone().requires_grad_(True)
        (g,) = torch.autograd.grad(call(op, {**given, name: torch._neg_view(leaf)}, "silu"), leaf, dy)
        other = given[name].detach().clone().requires_grad_(True)
        (h,) = torch.autograd.grad(call(op, {**given, name: -other}, "silu"), other, dy)
        assert torch.equal(g.resolve_neg(), h.resolve_neg())
    t = {k: v.detach().clone() for k, v in given.items()}
    t["x"].requires_grad_(True)
    (g,) = torch.autograd.grad(call(op, t, "silu"), t["x"], torch._neg_view(dy))
    (h,) = torch.autograd.grad(call(op, t, "silu"), t["x"], -dy)
    assert torch.equal(g, h)
