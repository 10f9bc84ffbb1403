"""Timed cases of the blocks around the products: linear layers, layer normalisation, products grouped by expert.

A case is a dict of plain values.  ``listed()`` names twelve, ``draw(rng)`` gives one more of the same ranges, ``prepare``
makes on the GPU what a program holds before the call, ``run`` is the one pass, ``work`` the bytes and operations it cannot
do without, ``exact`` the result from the definition in 64 bits.  With ``own`` false ``run`` computes the operators from
elementary torch operations in 32 bits, with ``own`` true through the library's public entry points.

    linear          y = act(x w + bias) + residual               x[m, k], w[k, n]
    layer_norm      y = (x - mean) / sqrt(var + eps) * weight + bias, mean and variance of a row
    grouped_matmul  y[r] = x[r] w[g] for the rows r of group g    offsets[g] <= r < offsets[g + 1]; other rows are zero

The ranges: linear layers of 1 to 8192 rows, n and k from 64 to 16384, with and without bias, activation and residual;
normalised rows of 16 to 32768 elements, 1 to 65536 of them; grouped products of 1 to 32768 rows in 1 to 128 groups, n and
k from 64 to 4096.  Each with and without its gradients, in bfloat16, float16 and float32.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZES = {"bf16": 2, "f16": 2, "f32": 4}
DEVICE = "cuda"
EPS = 1e-5

MOST_FLOPS = 6.0 * 8192 * 4096 * 4096
MOST_ELEMENTS = 16384 * 8192
MOST_WEIGHTS = 1 << 28


def listed():
    return [
        # one token's output projection, added to the residual stream: the weight is streamed once
        dict(name="linear_token", op="linear", m=1, n=4096, k=4096, dtype="bf16", layout="nt", bias=True, act="none", residual=True, train=False),
        # a decode batch through an up-projection
        dict(name="linear_batch", op="linear", m=48, n=14336, k=4096, dtype="f16", layout="nn", bias=True, act="silu", residual=False, train=False),
        # sizes that no tile divides, in 32 bits
        dict(name="linear_ragged", op="linear", m=333, n=1001, k=700, dtype="f32", layout="nn", bias=True, act="gelu", residual=True, train=False),
        # a training step of a small layer of odd sizes
        dict(name="linear_train_small", op="linear", m=1025, n=770, k=514, dtype="f16", layout="nt", bias=True, act="relu", residual=True, train=True),
        # a training step of a large up-projection: output and the gradients of input, weight and bias
        dict(name="linear_train", op="linear", m=8192, n=4096, k=4096, dtype="bf16", layout="nn", bias=True, act="gelu_tanh", residual=False, train=True),
        # one token's row
        dict(name="norm_token", op="norm", rows=1, n=4096, dtype="bf16", weight=True, bias=True, train=False),
        # an odd batch in 32 bits with its gradients
        dict(name="norm_ragged", op="norm", rows=1023, n=1501, dtype="f32", weight=True, bias=True, train=True),
        # a training batch: output and the gradients of input, weight and bias
        dict(name="norm_train", op="norm", rows=16384, n=8192, dtype="bf16", weight=True, bias=True, train=True),
        # eight tokens to two experts each of 64
        dict(name="grouped_decode", op="grouped", rows=16, groups=64, k=4096, n=2048, dtype="bf16", layout="nn", train=False),
        # a prompt, transposed weights of a checkpoint
        dict(name="grouped_prompt", op="grouped", rows=8192, groups=64, k=2048, n=2816, dtype="f16", layout="nt", train=False),
        # odd sizes and an odd number of groups with the gradients, in 32 bits
        dict(name="grouped_ragged", op="grouped", rows=1537, groups=7, k=390, n=517, dtype="f32", layout="nn", train=True),
        # a training batch: output and the gradients of rows and weights
        dict(name="grouped_train", op="grouped", rows=32768, groups=32, k=2048, n=2048, dtype="bf16", layout="nn", train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size of the range: half of them as they fall, odd ones among them, half in whole blocks of 32."""
    v = _log(rng, lo, hi)
    return v if rng.random() < 0.5 else max(lo, v // 32 * 32)


def draw(rng):
    while True:
        op = rng.choice(["linear", "linear", "norm", "grouped", "grouped"])
        dtype = rng.choice(["bf16", "bf16", "f16", "f16", "f32"])
        train = rng.random() < 0.5
        if op == "linear":
            # (32 bits and a gradient: no relu, whose derivative jumps where a sum's last bit decides)
            acts = ["none", "gelu", "gelu_tanh", "silu"] + ([] if dtype == "f32" and train else ["relu"])
            case = dict(op=op, m=_log(rng, 1, 8192), n=_size(rng, 64, 16384), k=_size(rng, 64, 16384), dtype=dtype, layout=rng.choice(["nn", "nt"]),
                        bias=rng.random() < 0.7, act=rng.choice(acts), residual=rng.random() < 0.5, train=train)
        elif op == "norm":
            weight = rng.random() < 0.8
            case = dict(op=op, rows=_log(rng, 1, 65536), n=_size(rng, 16, 32768), dtype=dtype, weight=weight, bias=weight and rng.random() < 0.7, train=train)
            if case["rows"] * case["n"] > MOST_ELEMENTS:
                continue
        else:
            case = dict(op=op, rows=_log(rng, 1, 32768), groups=rng.choice([1, 2, 4, 7, 8, 16, 32, 60, 64, 128]), k=_size(rng, 64, 4096),
                        n=_size(rng, 64, 4096), dtype=dtype, layout=rng.choice(["nn", "nt"]), train=train)
            if case["groups"] * case["k"] * case["n"] > MOST_WEIGHTS:
                continue
        if work(case)["flops"] <= MOST_FLOPS:
            return case


def work(case):
    es = SIZES[case["dtype"]]
    train = case["train"]
    if case["op"] == "linear":
        # forward: x, w, bias and residual in, y out; backward: dy in, the gradients out (x and w may still be in the caches)
        m, n, k = case["m"], case["n"], case["k"]
        b = (m * k + k * n + m * n + (n if case["bias"] else 0) + (m * n if case["residual"] else 0)) * es
        if train:
            b += (m * n + m * k + k * n + (n if case["bias"] else 0)) * es
        return {"bytes": float(b), "flops": (6.0 if train else 2.0) * m * n * k}
    if case["op"] == "norm":
        r, n = case["rows"], case["n"]
        params = (n if case["weight"] else 0) + (n if case["bias"] else 0)
        b = (2 * r * n + params) * es
        if train:
            b += (2 * r * n + params) * es
        return {"bytes": float(b), "flops": (20.0 if train else 8.0) * r * n}
    r, g, k, n = case["rows"], case["groups"], case["k"], case["n"]
    active = g * (1.0 - (1.0 - 1.0 / g) ** r)
    b = (r * k + active * k * n + r * n) * es + 4 * (g + 1)
    if train:
        b += (r * n + r * k + g * k * n) * es
    return {"bytes": float(b), "flops": (6.0 if train else 2.0) * r * n * k}


# ---------------------------------------------------------------------------------------------------------------- inputs
def _activations(rows, cols, dtype, g):
    """Activations with channels of different strength, as the layers of a trained model have them."""
    channel = torch.exp(0.5 * torch.randn(cols, device=DEVICE, generator=g))
    return (torch.randn(rows, cols, device=DEVICE, generator=g) * channel).to(dtype)


def _inputs(case, seed):
    g = torch.Generator(DEVICE)
    g.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    normal = lambda *shape: torch.randn(*shape, device=DEVICE, generator=g)  # noqa: E731
    s = {"case": case}
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        s["x"] = _activations(m, k, dtype, g)
        s["w"] = (normal(k, n) / math.sqrt(k)).to(dtype) if case["layout"] == "nn" else (normal(n, k) / math.sqrt(k)).to(dtype).t()
        if case["bias"]:
            s["bias"] = (0.5 * normal(n)).to(dtype)
        if case["residual"]:
            s["residual"] = normal(m, n).to(dtype)
        shape = (m, n)
    elif case["op"] == "norm":
        r, n = case["rows"], case["n"]
        s["x"] = (_activations(r, n, torch.float32, g) + 0.3 * normal(r, 1)).to(dtype)
        if case["weight"]:
            s["weight"] = (1.0 + 0.2 * normal(n)).to(dtype)
        if case["bias"]:
            s["bias"] = (0.2 * normal(n)).to(dtype)
        shape = (r, n)
    else:
        r, e, k, n = case["rows"], case["groups"], case["k"], case["n"]
        # rows of an uneven router, sorted by group; a few rows behind the last group belong to none, as empty slots do
        popular = torch.softmax(0.4 * normal(e), dim=0)
        group = torch.multinomial(popular, r, replacement=True, generator=g)
        group = torch.where(torch.rand(r, device=DEVICE, generator=g) < 0.02, e, group)
        counts = (group.unsqueeze(0) == torch.arange(e, device=DEVICE).unsqueeze(1)).sum(dim=1)
        s["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
        s["x"] = _activations(r, k, dtype, g)
        s["w"] = (normal(e, k, n) / math.sqrt(k)).to(dtype) if case["layout"] == "nn" else (normal(e, n, k) / math.sqrt(k)).to(dtype).transpose(1, 2)
        shape = (r, n)
    if case["train"]:
        s["dy"] = normal(*shape).to(dtype)
    return s


_LEAVES = {"linear": ("x", "w", "bias", "residual"), "norm": ("x", "weight", "bias"), "grouped": ("x", "w")}


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and case["train"]:
        for name in _LEAVES[case["op"]]:
            if name in s:
                s[name].requires_grad_(True)
    return s


# ---------------------------------------------------------------------------------------------------------------- the pass
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    import tritonix

    case = s["case"]
    if case["op"] == "linear":
        y = tritonix.linear(s["x"], s["w"], s.get("bias"), activation=None if case["act"] == "none" else case["act"], residual=s.get("residual"))
    elif case["op"] == "norm":
        y = tritonix.layer_norm(s["x"], s.get("weight"), s.get("bias"), eps=EPS)
    else:
        y = tritonix.grouped_matmul(s["x"], s["w"], s["offsets"])
    if not case["train"]:
        return {"y": y}
    names = [name for name in _LEAVES[case["op"]] if name in s]
    grads = torch.autograd.grad(y, [s[name] for name in names], s["dy"])
    return {"y": y.detach(), **{"d" + name: grad for name, grad in zip(names, grads)}}


def _act_plain(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def _act_slope_plain(z, act):
    if act == "relu":
        return (z > 0).float()
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    t = torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z))
    return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * math.sqrt(2.0 / math.pi) * (1.0 + 3.0 * 0.044715 * z * z)


def _linear_plain(s):
    case = s["case"]
    dtype = s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    z = x @ w
    if case["bias"]:
        z = z + s["bias"].float()
    y = _act_plain(z, case["act"])
    if case["residual"]:
        y = y + s["residual"].float()
    out = {"y": y.to(dtype)}
    if case["train"]:
        dz = s["dy"].float()
        if case["act"] != "none":
            dz = dz * _act_slope_plain(z, case["act"])
        out["dx"] = (dz @ w.t()).to(dtype)
        out["dw"] = (x.t() @ dz).to(dtype)
        if case["bias"]:
            out["dbias"] = dz.sum(dim=0).to(dtype)
        if case["residual"]:
            out["dresidual"] = s["dy"]
    return out


def _norm_plain(s):
    case = s["case"]
    dtype = s["x"].dtype
    x = s["x"].float()
    centred = x - x.mean(dim=1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(dim=1, keepdim=True) + EPS)
    unit = centred * rstd
    y = unit
    if case["weight"]:
        y = y * s["weight"].float()
    if case["bias"]:
        y = y + s["bias"].float()
    out = {"y": y.to(dtype)}
    if case["train"]:
        dy = s["dy"].float()
        g = dy * s["weight"].float() if case["weight"] else dy
        out["dx"] = (rstd * (g - g.mean(dim=1, keepdim=True) - unit * (g * unit).mean(dim=1, keepdim=True))).to(dtype)
        if case["weight"]:
            out["dweight"] = (dy * unit).sum(dim=0).to(dtype)
        if case["bias"]:
            out["dbias"] = dy.sum(dim=0).to(dtype)
    return out


def _grouped_plain(s):
    """The groups that have rows, padded to the longest of them: one batch of products."""
    case = s["case"]
    dtype = s["x"].dtype
    offsets = s["offsets"].long()
    counts = offsets[1:] - offsets[:-1]
    used = torch.nonzero(counts).squeeze(1)
    out = {"y": torch.zeros(case["rows"], case["n"], dtype=dtype, device=s["x"].device)}
    if case["train"]:
        out["dx"], out["dw"] = torch.zeros_like(s["x"]), torch.zeros_like(s["w"])
    if used.numel() == 0:
        return out
    longest = int(counts.max())
    place = torch.arange(longest, device=offsets.device)
    here = place < counts[used].unsqueeze(1)
    rows = torch.where(here, offsets[used].unsqueeze(1) + place, 0)
    at = rows[here]
    x = torch.where(here.unsqueeze(2), s["x"].float()[rows], torch.zeros((), device=rows.device))
    w = s["w"][used].float().contiguous()
    out["y"][at] = torch.bmm(x, w)[here].to(dtype)
    if case["train"]:
        dy = torch.where(here.unsqueeze(2), s["dy"].float()[rows], torch.zeros((), device=rows.device))
        out["dx"][at] = torch.bmm(dy, w.transpose(1, 2).contiguous())[here].to(dtype)
        out["dw"][used] = torch.bmm(x.transpose(1, 2).contiguous(), dy).to(dtype)
    return out


def _run_plain(s):
    return {"linear": _linear_plain, "norm": _norm_plain, "grouped": _grouped_plain}[s["case"]["op"]](s)


# ---------------------------------------------------------------------------------------------------------------- 64 bits
def _exact_linear(case, s):
    names = [name for name in _LEAVES["linear"] if name in s]
    v = {name: s[name].detach().double().requires_grad_(case["train"]) for name in names}
    z = torch.matmul(v["x"], v["w"])
    if "bias" in v:
        z = torch.add(z, v["bias"])
    f = torch.nn.functional
    y = {"none": lambda t: t, "relu": f.relu, "silu": f.silu, "gelu": f.gelu, "gelu_tanh": lambda t: f.gelu(t, approximate="tanh")}[case["act"]](z)
    if "residual" in v:
        y = torch.add(y, v["residual"])
    out = {"y": y.detach()}
    if case["train"]:
        grads = torch.autograd.grad(y, [v[name] for name in names], s["dy"].double())
        out.update({"d" + name: grad for name, grad in zip(names, grads)})
    return out


def _exact_norm(case, s):
    names = [name for name in _LEAVES["norm"] if name in s]
    v = {name: s[name].detach().double().requires_grad_(case["train"]) for name in names}
    var, mean = torch.var_mean(v["x"], dim=1, correction=0, keepdim=True)
    y = torch.div(torch.sub(v["x"], mean), torch.sqrt(var + EPS))
    if "weight" in v:
        y = torch.mul(y, v["weight"])
    if "bias" in v:
        y = torch.add(y, v["bias"])
    out = {"y": y.detach()}
    if case["train"]:
        grads = torch.autograd.grad(y, [v[name] for name in names], s["dy"].double())
        out.update({"d" + name: grad for name, grad in zip(names, grads)})
    return out


def _exact_grouped(case, s):
    x, w = s["x"].double(), s["w"]
    bounds = s["offsets"].tolist()
    out = {"y": torch.zeros(case["rows"], case["n"], dtype=torch.float64, device=x.device)}
    if case["train"]:
        dy = s["dy"].double()
        out["dx"] = torch.zeros_like(x)
        out["dw"] = torch.zeros(case["groups"], case["k"], case["n"], dtype=torch.float64, device=x.device)
    for g, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
        if lo < hi:
            one = w[g].double()
            out["y"][lo:hi] = x[lo:hi].mm(one)
            if case["train"]:
                out["dx"][lo:hi] = dy[lo:hi].mm(one.t())
                out["dw"][g] = x[lo:hi].t().mm(dy[lo:hi])
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    return {"linear": _exact_linear, "norm": _exact_norm, "grouped": _exact_grouped}[case["op"]](case, s)
