"""Definitions in 64 bits of linear layers, layer normalisation and grouped products, each with a bound on the error of a computation that holds
sums in 32 bits and rounds its results once.

Bounds are to first order, elementwise, from: half a step of a type, u = eps / 2, relative to a rounded value (and half the smallest subnormal);
E = 2^-23 for one operation in 32 bits, twice half a step, since the matrix instruction's inner sums round in a way of their own; a sum of t terms
in 32 bits t E times the sum of magnitudes; float32 products by heads and tails 3.5 * 2^-18 of the sum of magnitudes beside it (a head is off by at most 2^-9 of the
operand and a tail by 2^-9 of that, for each operand, and the product of the tails is left out)."""
import math

import torch

E = 2.0 ** -23
SPLIT = 3.5 * 2.0 ** -18
F = torch.float64


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def rounding(value, dtype):
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}[dtype]
    return unit(dtype) * value.abs() + tiny


def activation(z, act):
    f = torch.nn.functional
    return {None: lambda t: t, "relu": f.relu, "silu": f.silu, "gelu": f.gelu, "gelu_tanh": lambda t: f.gelu(t, approximate="tanh")}[act](z)


def slope(z, act):
    if act is None:
        return torch.ones_like(z)
    if act == "relu":
        return (z > 0).to(z.dtype)
    z = z.detach().requires_grad_(True)
    with torch.enable_grad():
        return torch.autograd.grad(activation(z, act).sum(), z)[0]


# largest |act'| (the value's error grows by at most it) and |act''| (the slope's)
STEEP = {None: 1.0, "relu": 1.0, "silu": 1.1, "gelu": 1.13, "gelu_tanh": 1.13}
BENT = {None: 0.0, "relu": 0.0, "silu": 0.5, "gelu": 0.8, "gelu_tanh": 0.85}


def product_error(a, b, dtype):
    """Of a @ b in 32 bits: the magnitudes' product, times the sum's share (and the split's)."""
    mags = a.abs() @ b.abs()
    return mags * ((a.shape[-1] + 2) * E + (SPLIT if dtype == torch.float32 else 0.0))


def linear(x, w, bias=None, act=None, residual=None, dy=None):
    """{name: (value, bound)} of y and, with dy, of the gradients."""
    dtype = x.dtype
    x, w = x.detach().to(F).cpu(), w.detach().to(F).cpu()
    bias64 = None if bias is None else bias.detach().to(F).cpu()
    z = x @ w
    ez = product_error(x, w, dtype)
    if bias is not None:
        z = z + bias64
        ez = ez + E * (z.abs() + bias64.abs())
    y = activation(z, act)
    # (the activation's own arithmetic: a dozen operations on numbers of z's size; __expf is good to 2 + |z| half steps of its argument)
    ey = STEEP[act] * ez + (0.0 if act in (None, "relu") else (12 + z.abs()) * E * z.abs())
    if residual is not None:
        r = residual.detach().to(F).cpu()
        y = y + r
        ey = ey + E * (y.abs() + r.abs())
    out = {"y": (y, ey + rounding(y, dtype))}
    if dy is None:
        return out
    g = dy.detach().to(F).cpu()
    s = slope(z, act)
    # the slope is taken at z as it was kept, rounded
    es = BENT[act] * (ez + rounding(z, dtype)) + (0.0 if act in (None, "relu") else (16 + z.abs()) * E * (1 + z.abs()))
    if act == "relu":
        es = (z.abs() <= ez + rounding(z, dtype)).to(F)
    dz = g * s
    edz = g.abs() * es + E * dz.abs()
    if bias is not None:
        db = dz.sum(dim=0)
        out["dbias"] = (db, edz.sum(dim=0) + x.shape[0] * E * dz.abs().sum(dim=0) + rounding(db, bias.dtype))
    kept = edz + (rounding(dz, dtype) if act is not None else 0.0)
    dx, dw = dz @ w.t(), x.t() @ dz
    out["dx"] = (dx, kept @ w.t().abs() + product_error(dz, w.t(), dtype) + rounding(dx, dtype))
    out["dw"] = (dw, x.t().abs() @ kept + product_error(x.t(), dz, dtype) + rounding(dw, dtype))
    if residual is not None:
        out["dresidual"] = (g, torch.zeros_like(g))
    return out


def layer_norm(x, weight=None, bias=None, eps=1e-5, dy=None):
    dtype = x.dtype
    x = x.detach().to(F).cpu()
    rows, n = x.shape
    w = torch.ones(n, dtype=F) if weight is None else weight.detach().to(F).cpu()
    b = torch.zeros(n, dtype=F) if bias is None else bias.detach().to(F).cpu()
    terms = n / 1024 + 96                  # additions on a row's longest way: a thread's own, then a tree
    mean = x.mean(dim=1, keepdim=True)
    c = x - mean
    var = (c * c).mean(dim=1, keepdim=True)
    rstd = 1.0 / torch.sqrt(var + eps)
    u = c * rstd
    emean = terms * E * x.abs().mean(dim=1, keepdim=True)
    ec = emean + E * (c.abs() + mean.abs())
    evar = 2 * (c.abs() * ec).mean(dim=1, keepdim=True) + (ec * ec).mean(dim=1, keepdim=True) + terms * E * var
    err = 0.5 * evar * rstd * rstd + 4 * E                 # of rstd, relative
    eu = ec * rstd + u.abs() * err + E * u.abs()
    y = u * w + b
    out = {"y": (y, eu * w.abs() + 3 * E * ((u * w).abs() + b.abs()) + rounding(y, dtype))}
    if dy is None:
        return out
    d = dy.detach().to(F).cpu()
    g = d * w
    a, s = g.mean(dim=1, keepdim=True), (g * u).mean(dim=1, keepdim=True)
    ea = (terms + 2) * E * g.abs().mean(dim=1, keepdim=True)
    es = (terms + 3) * E * (g * u).abs().mean(dim=1, keepdim=True) + (g.abs() * eu).mean(dim=1, keepdim=True)
    inner = g - a - u * s
    dx = rstd * inner
    edx = rstd * (ea + u.abs() * es + s.abs() * eu + 4 * E * (g.abs() + a.abs() + (u * s).abs())) + dx.abs() * err
    out["dx"] = (dx, edx + rounding(dx, dtype))
    if weight is not None:
        dw = (d * u).sum(dim=0)
        out["dweight"] = (dw, (d.abs() * eu).sum(dim=0) + (rows + 2) * E * (d * u).abs().sum(dim=0) + rounding(dw, weight.dtype))
    if bias is not None:
        db = d.sum(dim=0)
        out["dbias"] = (db, (rows + 2) * E * d.abs().sum(dim=0) + rounding(db, bias.dtype))
    return out


def bounds_of(offsets, rows):
    """Group bounds as the operator takes them: inside [0, rows], not decreasing."""
    out, top = [], 0
    for v in offsets:
        top = max(top, min(max(int(v), 0), rows))
        out.append(top)
    return out


def grouped(x, w, offsets, dy=None):
    dtype = x.dtype
    x, w = x.detach().to(F).cpu(), w.detach().to(F).cpu()
    rows, n = x.shape[0], w.shape[2]
    at = bounds_of(offsets.tolist(), rows)
    share = lambda t: (t + 2) * E  # noqa: E731
    y, ey = torch.zeros(rows, n, dtype=F), torch.zeros(rows, n, dtype=F)
    dx, edx, dw, edw = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(w)
    g = None if dy is None else dy.detach().to(F).cpu()
    for e, (lo, hi) in enumerate(zip(at, at[1:])):
        if lo == hi:
            continue
        y[lo:hi] = x[lo:hi] @ w[e]
        ey[lo:hi] = share(x.shape[1]) * (x[lo:hi].abs() @ w[e].abs())
        if g is not None:
            dx[lo:hi] = g[lo:hi] @ w[e].t()
            edx[lo:hi] = share(n) * (g[lo:hi].abs() @ w[e].t().abs())
            dw[e] = x[lo:hi].t() @ g[lo:hi]
            edw[e] = share(hi - lo) * (x[lo:hi].t().abs() @ g[lo:hi].abs())
    out = {"y": (y, ey + rounding(y, dtype))}
    if g is not None:
        out["dx"], out["dw"] = (dx, edx + rounding(dx, dtype)), (dw, edw + rounding(dw, dtype))
    return out


def check(name, got, wanted, dtype=None):
    """``got`` within its bound of the definition, everywhere; the text says where it is not."""
    value, bound = wanted
    if dtype is not None:
        assert got.dtype == dtype, (name, got.dtype)
    assert tuple(got.shape) == tuple(value.shape), (name, tuple(got.shape), tuple(value.shape))
    got = got.detach().to(F).cpu()
    off = (got - value).abs()
    bad = ~(off <= bound)
    if bool(bad.any()):
        i = int(torch.where(bad.flatten(), off.flatten() / (bound.flatten() + 1e-300), torch.zeros(())).nan_to_num(math.inf).argmax())
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} out of bounds, worst at {i}: got {got.flatten()[i]}, definition "
                             f"{value.flatten()[i]}, bound {bound.flatten()[i]}")


def draw(device, *shape, dtype=torch.bfloat16, seed=0, scale=1.0):
    g = torch.Generator("cpu").manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(device)
