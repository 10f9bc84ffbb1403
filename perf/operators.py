"""Timed cases of the 4-bit microscaled products and of the mixture of experts built on them.

A case is a dict of plain values.  ``listed()`` names twelve, ``draw(rng)`` gives one more of the same ranges, ``prepare``
makes on the GPU what a program holds before the call, ``run`` is the one pass, ``work`` the bytes and operations it cannot
do without, ``exact`` the result from the definition in 64 bits.  With ``own`` false ``run`` computes the operators from
elementary torch operations in 32 bits, with ``own`` true through the library's public entry points.

The ranges: quantisation of 1 to 8192 rows of 32 to 28672 elements along either dimension; products of 1 to 8192 rows, n and
k from 64 to 16384; training steps of linear layers of 32 to 8192 rows over widths 64 to 4096; routing of 1 to 65536 tokens
to 8 to 512 experts; experts' products of 1 to 8192 tokens, widths 128 to 4096, 4 to 128 experts, 1 to 8 of them a token.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZES = {"bf16": 2, "f16": 2, "f32": 4}
DEVICE = "cuda"
MX_BYTES = 17.0 / 32.0          # one element of a microscaled tensor: half a byte, and a scale byte for 32

MOST_FLOPS = 2.0 * 8192 ** 3
MOST_ELEMENTS = 8192 * 28672
MOST_WEIGHTS = 64 * 4096 * 2048


def listed():
    return [
        # one token of a decoder: 256 experts in 8 groups, chosen by sigmoid scores with a balance bias
        dict(name="route_token", op="route", t=1, e=256, k=8, dtype="f32", scoring="sigmoid", bias=True, groups=8, top_groups=4,
             group_top=2, renorm=True, scale=2.5, masked=False, train=False),
        # a ragged prompt in bfloat16; padding rows and switched-off experts carry -inf
        dict(name="route_prompt", op="route", t=4099, e=60, k=6, dtype="bf16", scoring="softmax", bias=False, groups=1, top_groups=1,
             group_top=1, renorm=False, scale=1.0, masked=True, train=False),
        # a training batch: the choice, and the gradient of the logits
        dict(name="route_train", op="route", t=65536, e=128, k=8, dtype="f32", scoring="softmax", bias=False, groups=1, top_groups=1,
             group_top=1, renorm=True, scale=1.0, masked=False, train=True),
        # an odd activation in float32, quantised down its columns (as the weight gradient's product takes it), and back
        dict(name="quantize_columns", op="quantize", rows=1001, cols=4100, dim=0, dtype="f32"),
        # a whole up-projection weight of the feed-forward block: the largest quantisation, and back
        dict(name="quantize_weight", op="quantize", rows=8192, cols=28672, dim=1, dtype="bf16"),
        # one token through a down-projection: the weight is streamed once
        dict(name="matmul_token", op="matmul", m=1, n=4096, k=14336, dtype="bf16"),
        # sizes that no tile divides
        dict(name="matmul_ragged", op="matmul", m=1025, n=2050, k=4100, dtype="f16"),
        # the large square product
        dict(name="matmul_large", op="matmul", m=8192, n=8192, k=8192, dtype="bf16"),
        # a training step of a linear layer: output, gradient of the input, gradient of the weight
        dict(name="linear_train", op="linear", m=8192, n=4096, k=4096, dtype="bf16"),
        # one token through the gated up-projections of its 8 experts
        dict(name="experts_up_token", op="up", t=1, e=64, k=8, d=4096, f=1024, dtype="bf16", holes=False),
        # a decode batch through the down-projections, joined with the routing weights; some slots are empty
        dict(name="experts_down_batch", op="down", t=64, e=64, k=8, d=4096, f=1024, dtype="bf16", holes=True),
        # a prompt of 8192 tokens through the up-projections: the largest call
        dict(name="experts_up_prompt", op="up", t=8192, e=64, k=8, d=4096, f=1024, dtype="bf16", holes=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size of the range: half of them as they fall, odd ones among them, half in whole blocks of 32."""
    v = _log(rng, lo, hi)
    return v if rng.random() < 0.5 else max(lo, v // 32 * 32)


def draw(rng):
    while True:
        op = rng.choice(["route", "quantize", "matmul", "matmul", "linear", "up", "up", "down"])
        dtype = rng.choice(["bf16", "f16"])
        if op == "route":
            e = rng.choice([8, 16, 60, 64, 96, 128, 160, 256, 384, 512])
            scoring = rng.choice(["softmax", "sigmoid"])
            bias = scoring == "sigmoid" and rng.random() < 0.7
            groups = rng.choice([1, 4, 8]) if e % 8 == 0 else 1
            top_groups = max(1, groups // 2)
            k = min(rng.choice([1, 2, 4, 6, 8]), e // groups * top_groups)
            train = rng.random() < 0.5
            case = dict(op=op, t=_log(rng, 1, 65536 * 128 // max(e, 128)), e=e, k=k, dtype=rng.choice(["f32", "bf16", "f16"]), scoring=scoring, bias=bias,
                        groups=groups, top_groups=top_groups, group_top=2 if bias else 1, renorm=rng.random() < 0.7,
                        scale=rng.choice([1.0, 2.5]), masked=rng.random() < 0.3, train=train)
        elif op == "quantize":
            case = dict(op=op, rows=_size(rng, 1, 8192), cols=_size(rng, 32, 28672), dim=rng.choice([0, 1]),
                        dtype=rng.choice(["bf16", "f16", "f32"]))
        elif op == "matmul":
            case = dict(op=op, m=_log(rng, 1, 8192), n=_size(rng, 64, 16384), k=_size(rng, 64, 16384), dtype=dtype)
        elif op == "linear":
            case = dict(op=op, m=_size(rng, 32, 8192), n=_size(rng, 64, 4096), k=_size(rng, 64, 4096), dtype=dtype)
        else:
            e = rng.choice([4, 8, 16, 32, 60, 64, 128])
            case = dict(op=op, t=_log(rng, 1, 8192), e=e, k=rng.choice([1, 2, 4, 6, 8]) if e >= 8 else 2, d=_size(rng, 128, 4096),
                        f=_size(rng, 128, 2048), dtype=dtype, holes=rng.random() < 0.3)
            if e * case["d"] * case["f"] * 2 > MOST_WEIGHTS * 2:
                continue
        if work(case)["flops"] <= MOST_FLOPS:
            return case


def work(case):
    op = case["op"]
    es = SIZES[case["dtype"]]
    if op == "route":
        # logits in; weights, experts, order and rows out, and the experts' offsets; training: logits and the weights'
        # gradient in, the logits' gradient out
        t, e, k = case["t"], case["e"], case["k"]
        b = t * e * es + t * k * 16 + 4 * (e + 1) + (4 * e if case["bias"] else 0)
        if case["train"]:
            b += 2 * t * e * es + t * k * 4
        return {"bytes": float(b), "flops": float(t * e * (4 + k) + (t * e * 4 if case["train"] else 0))}
    if op == "quantize":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (es + 2 * MX_BYTES + es), "flops": 6.0 * n}
    if op == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k * es + n * k * MX_BYTES + m * n * es, "flops": 2.0 * m * n * k}
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": float(2 * m * k + 2 * k * n + 2 * m * n) * es, "flops": 6.0 * m * n * k}
    t, e, k, d, f = (case[v] for v in ("t", "e", "k", "d", "f"))
    active = e * (1.0 - (1.0 - k / e) ** t)
    if op == "up":
        return {"bytes": t * d * es + active * d * 2 * f * MX_BYTES + t * k * f * es, "flops": 4.0 * t * k * d * f}
    return {"bytes": t * k * f * es + active * d * f * MX_BYTES + t * d * es, "flops": 2.0 * t * k * d * f}


# ---------------------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(DEVICE)
    g.manual_seed(seed)
    return g


def _activations(rows, cols, dtype, g):
    """Activations with channels of different strength, as the layers of a trained model have them."""
    channel = torch.exp(0.5 * torch.randn(cols, device=DEVICE, generator=g))
    return (torch.randn(rows, cols, device=DEVICE, generator=g) * channel).to(dtype)


def _mx_codes(w):
    """Rows of a float32 matrix as a checkpoint holds them: two 4-bit codes a byte, the even element in the low half,
    and a scale byte for 32 elements."""
    q, scale = _blocks_plain(w)
    mag = q.abs()
    code = torch.zeros(mag.shape, dtype=torch.uint8, device=w.device)
    for level in (0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0):
        code += mag >= level
    code += torch.signbit(q).to(torch.uint8) * 8
    n, k = w.shape
    code = code.reshape(n, -1)[:, :k]
    if k % 2:
        code = torch.cat([code, torch.zeros(n, 1, dtype=torch.uint8, device=w.device)], dim=1)
    codes = code[:, 0::2] + code[:, 1::2] * 16
    scales = (torch.frexp(scale.squeeze(-1)).exponent - 1 + 127).to(torch.uint8)
    return codes.contiguous(), scales.contiguous()


def _weights(n, k, g):
    return _mx_codes(torch.randn(n, k, device=DEVICE, generator=g) / math.sqrt(k))


def _logits(case, g):
    t, e = case["t"], case["e"]
    dtype = DTYPES[case["dtype"]]
    popular = 0.3 * torch.randn(e, device=DEVICE, generator=g)
    bias = 0.05 * torch.randn(e, device=DEVICE, generator=g) if case["bias"] else None
    x = (torch.randn(t, e, device=DEVICE, generator=g) + popular).to(dtype)
    if bias is not None:
        # Two experts whose biased scores agree to the last bits of an exponential are as good as each other, whichever an
        # implementation takes: such rows are drawn again, so that every row here has one answer.
        for _ in range(20):
            close = _close_rows(case, x, bias)
            if not bool(close.any()):
                break
            x[close] = (torch.randn(int(close.sum()), e, device=DEVICE, generator=g) + popular).to(dtype)
    if case["masked"]:
        off = torch.rand(t, e, device=DEVICE, generator=g) < 0.1
        off[torch.rand(t, device=DEVICE, generator=g) < 0.05] = True
        if bias is None:
            x[off] = -math.inf
        else:
            x[off.all(dim=1)] = -math.inf
    return x, bias


def _close_rows(case, x, bias):
    key = torch.sigmoid(x.double()) + bias.double()
    t, e = key.shape
    close = torch.zeros(t, dtype=torch.bool, device=x.device)
    groups = case["groups"]
    if groups > 1:
        score = key.view(t, groups, e // groups).topk(case["group_top"], dim=-1).values.sum(-1).sort(dim=1, descending=True).values
        close |= (score[:, :-1] - score[:, 1:]).amin(dim=1) < 1e-5
    kept = _kept_groups(key, case)
    ranked = key.masked_fill(~kept, -math.inf).sort(dim=1, descending=True).values
    gaps = (ranked[:, :-1] - ranked[:, 1:]).nan_to_num(1.0, posinf=1.0)
    return close | (gaps[:, :case["k"]].amin(dim=1) < 2e-6)


def _kept_groups(key, case):
    t, e = key.shape
    groups = case["groups"]
    score = key.view(t, groups, e // groups).topk(case["group_top"], dim=-1).values.sum(-1)
    best = score.sort(dim=1, descending=True, stable=True).indices[:, :case["top_groups"]]
    kept = torch.zeros(t, groups, dtype=torch.bool, device=key.device).scatter_(1, best, True)
    return kept.unsqueeze(-1).expand(t, groups, e // groups).reshape(t, e)


def _choice(case, g):
    """Tokens' experts and weights of an uneven router."""
    t, e, k = case["t"], case["e"], case["k"]
    logits = torch.randn(t, e, device=DEVICE, generator=g) + 0.5 * torch.randn(e, device=DEVICE, generator=g)
    top = logits.topk(k, dim=1)
    weights, experts = torch.softmax(top.values, dim=1), top.indices.to(torch.int32)
    if case["holes"]:
        hole = torch.rand(t, k, device=DEVICE, generator=g) < 0.1
        weights, experts = weights.masked_fill(hole, 0.0), experts.masked_fill(hole, -1)
    return weights.contiguous(), experts.contiguous()


def _inputs(case, seed):
    g = _gen(seed)
    op = case["op"]
    dtype = DTYPES[case["dtype"]]
    s = {"case": case}
    if op == "route":
        s["logits"], s["bias"] = _logits(case, g)
        s["grad"] = torch.randn(case["t"], case["k"], device=DEVICE, generator=g)
    elif op == "quantize":
        s["x"] = _activations(case["rows"], case["cols"], dtype, g)
    elif op == "matmul":
        s["x"] = _activations(case["m"], case["k"], dtype, g)
        s["codes"], s["scales"] = _weights(case["n"], case["k"], g)
    elif op == "linear":
        s["x"] = _activations(case["m"], case["k"], dtype, g)
        s["w"] = (torch.randn(case["k"], case["n"], device=DEVICE, generator=g) / math.sqrt(case["k"])).to(dtype)
        s["dy"] = torch.randn(case["m"], case["n"], device=DEVICE, generator=g).to(dtype)
    else:
        e, d, f = case["e"], case["d"], case["f"]
        s["weights"], s["experts"] = _choice(case, g)
        n, k = (2 * f, d) if op == "up" else (d, f)
        rows = case["t"] if op == "up" else case["t"] * case["k"]
        s["x"] = _activations(rows, k, dtype, g)
        made = [_weights(n, k, g) for _ in range(e)]
        s["codes"], s["scales"] = torch.stack([c for c, _ in made]), torch.stack([v for _, v in made])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        import tritonix

        if case["op"] in ("matmul", "up", "down"):
            # the weight of the checkpoint, laid out once
            s["w"] = tritonix.MXTensor.from_codes(s.pop("codes"), s.pop("scales"), case["d"] if case["op"] == "up" else
                                                  case["f"] if case["op"] == "down" else case["k"], dim=-2)
        if case["op"] in ("up", "down"):
            s["routing"] = tritonix.moe_plan(s["experts"], s["weights"], case["e"])
        if case["op"] == "linear":
            s["x"].requires_grad_(True)
            s["w"].requires_grad_(True)
    return s


# ---------------------------------------------------------------------------------------------------------------- the pass
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    import tritonix

    case = s["case"]
    op = case["op"]
    if op == "route":
        r = tritonix.moe_route(s["logits"], case["k"], scoring=case["scoring"], bias=s["bias"], num_groups=case["groups"],
                               top_groups=case["top_groups"], group_top=case["group_top"], renormalize=case["renorm"], scale=case["scale"])
        out = {"weights": r.weights, "experts": r.experts, "offsets": r.offsets, "order": r.order, "rows": r.rows}
        if case["train"]:
            out["grad"] = tritonix.moe_route_backward(s["grad"], s["logits"], r)
        return out
    if op == "quantize":
        return tritonix.mx_dequantize(tritonix.mx_quantize(s["x"], dim=case["dim"]), s["x"].dtype)
    if op == "matmul":
        return tritonix.mx_matmul(s["x"], s["w"])
    if op == "linear":
        y = tritonix.mx_linear(s["x"], s["w"])
        dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw}
    if op == "up":
        return tritonix.moe_glu(s["x"], s["w"], s["routing"])
    return tritonix.moe_down(s["x"], s["w"], s["routing"])


def _blocks_plain(x):
    """Rows cut into blocks of 32: the 4-bit values of each block and its scale, in 32 bits."""
    x = x.float()
    n, k = x.shape
    pad = -k % 32
    if pad:
        x = torch.cat([x, x.new_zeros(n, pad)], dim=1)
    x = x.view(n, -1, 32)
    amax = x.abs().amax(dim=-1, keepdim=True)
    e = (torch.frexp(amax).exponent - 3).masked_fill(amax == 0, 0).clamp(-127, 125)
    scale = torch.ldexp(torch.ones_like(amax), e)
    v = x / scale
    a = v.abs()
    # round to nearest on 0, 0.5, 1, 1.5, 2, 3, 4, 6, ties to the even code, 6 and above to 6
    q = 0.5 * ((a > 0.25).float() + (a >= 0.75).float() + (a > 1.25).float() + (a >= 1.75).float())
    q = q + (a > 2.5).float() + (a >= 3.5).float() + 2.0 * (a > 5.0).float()
    return torch.where(v < 0, -q, q), scale


def _quantized_plain(x, dim=1):
    if dim == 0:
        return _quantized_plain(x.t()).t()
    q, scale = _blocks_plain(x)
    return (q * scale).view(x.shape[0], -1)[:, :x.shape[1]]


def _values_plain(codes, scales, k):
    """What the codes of a weight stand for, in 32 bits."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=codes.device)
    pair = torch.stack([table[(codes & 15).int()], table[(codes >> 4).int()]], dim=-1)
    q = pair.reshape(codes.shape[0], -1)[:, :k]
    scale = torch.ldexp(torch.ones((), device=codes.device), scales.int() - 127)
    return q * scale.repeat_interleave(32, dim=1)[:, :k]


def _plan_plain(experts, num_experts):
    """Pairs of token and slot in the order of their experts, and where each pair went; empty slots have no place."""
    flat = experts.reshape(-1)
    placed = flat >= 0
    order = torch.sort(torch.where(placed, flat, num_experts), stable=True).indices
    counts = (flat.unsqueeze(0) == torch.arange(num_experts, device=flat.device).unsqueeze(1)).sum(dim=1)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    total = offsets[-1]
    place = torch.arange(flat.numel(), device=flat.device)
    rows = torch.empty_like(place)
    rows[order] = torch.where(place < total, place, -1)
    order = torch.where(place < total, order, -1)
    return offsets.int(), order.int(), rows.view_as(experts).int()


def _route_plain(s):
    case = s["case"]
    x = s["logits"].float()
    t, e = x.shape
    if case["scoring"] == "softmax":
        p = torch.exp(x - x.amax(dim=1, keepdim=True))
        p = p / p.sum(dim=1, keepdim=True)
        p = torch.where(x == -math.inf, torch.zeros_like(p), p)
    else:
        p = 1.0 / (1.0 + torch.exp(-x))
    key = x if s["bias"] is None else torch.where(x == -math.inf, x, p + s["bias"])
    groups = case["groups"]
    if groups > 1:
        top = key.view(t, groups, e // groups).sort(dim=-1, descending=True).values[..., :case["group_top"]]
        best = top.sum(dim=-1).sort(dim=1, descending=True, stable=True).indices[:, :case["top_groups"]]
        kept = (best.unsqueeze(-1) == torch.arange(groups, device=x.device)).any(dim=1)
        key = torch.where(kept.repeat_interleave(e // groups, dim=1), key, torch.full_like(key, -math.inf))
    values, experts = key.sort(dim=1, descending=True, stable=True)
    values, experts = values[:, :case["k"]], experts[:, :case["k"]]
    chosen = values > -math.inf
    score = torch.where(chosen, p.gather(1, experts), torch.zeros_like(values))
    total = score.sum(dim=1, keepdim=True)
    total = torch.where(total > 0, total, torch.ones_like(total))
    weights = case["scale"] * (score / total if case["renorm"] else score)
    experts32 = torch.where(chosen, experts, -1).int()
    offsets, order, rows = _plan_plain(experts32, e)
    out = {"weights": weights, "experts": experts32, "offsets": offsets, "order": order, "rows": rows}
    if case["train"]:
        g = torch.where(chosen, s["grad"], torch.zeros_like(score))
        if case["renorm"]:
            share = score / total
            ds = case["scale"] * (g - (share * g).sum(dim=1, keepdim=True)) / total
        else:
            ds = case["scale"] * g
        ds = torch.where(chosen, ds, torch.zeros_like(ds))
        if case["scoring"] == "softmax":
            dl = -p * (score * ds).sum(dim=1, keepdim=True)
            dl = dl.scatter_add(1, experts, score * ds)
        else:
            dl = torch.zeros_like(p).scatter_add(1, experts, ds * score * (1.0 - score))
        out["grad"] = dl.to(s["logits"].dtype)
    return out


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op == "route":
        return _route_plain(s)
    dtype = s["x"].dtype
    if op == "quantize":
        return _quantized_plain(s["x"], case["dim"]).to(dtype)
    if op == "matmul":
        return (_quantized_plain(s["x"]) @ _values_plain(s["codes"], s["scales"], case["k"]).t()).to(dtype)
    if op == "linear":
        x, w, dy = s["x"], s["w"], s["dy"]
        y = _quantized_plain(x) @ _quantized_plain(w, 0)
        dx = _quantized_plain(dy) @ _quantized_plain(w).t()
        dw = _quantized_plain(x, 0).t() @ _quantized_plain(dy, 0)
        return {"y": y.to(dtype), "dx": dx.to(dtype), "dw": dw.to(dtype)}
    offsets, order, rows = _plan_plain(s["experts"], case["e"])
    xq = _quantized_plain(s["x"])
    bounds = offsets.tolist()
    t, k, d, f = case["t"], case["k"], case["d"], case["f"]
    h = torch.zeros(t * k, f if op == "up" else d, device=xq.device)
    for i in range(case["e"]):
        lo, hi = bounds[i], bounds[i + 1]
        if lo == hi:
            continue
        if op == "up":
            z = xq[order[lo:hi].long() // k] @ _values_plain(s["codes"][i], s["scales"][i], d).t()
            gate, linear = z[:, 0::2], z[:, 1::2]
            h[lo:hi] = gate / (1.0 + torch.exp(-gate)) * linear
        else:
            h[lo:hi] = xq[lo:hi] @ _values_plain(s["codes"][i], s["scales"][i], f).t()
    if op == "up":
        return h.to(dtype)
    taken = torch.where((rows >= 0).unsqueeze(-1), h[rows.clamp(min=0).long()], torch.zeros((), device=h.device))
    return (taken * s["weights"].unsqueeze(-1)).sum(dim=1).to(dtype)


# ---------------------------------------------------------------------------------------------------------------- 64 bits
def _exact_quantized(x):
    """Blocks of 32 along the last dimension, from the definition: the scale is the power of two two below the largest
    magnitude's, the grid's step half of the value's own power of two (at least 0.5), ties to the even multiple."""
    x = x.double()
    n, k = x.shape
    blocks = torch.nn.functional.pad(x, (0, -k % 32)).unflatten(1, (-1, 32))
    top = blocks.abs().max(dim=2, keepdim=True).values
    scale = torch.exp2(torch.floor(torch.log2(top.clamp(min=2.0 ** -125))).clamp(max=127) - 2)
    v = blocks / scale
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=1.0))) - 1)
    q = (torch.round(v / step) * step).clamp(-6, 6)
    return (q * scale).flatten(1)[:, :k]


def _exact_values(codes, scales, k):
    code = torch.stack([codes % 16, codes // 16], dim=2).flatten(1)[:, :k].double()
    sign = 1.0 - 2.0 * torch.floor(code / 8)
    exponent, mantissa = torch.floor(code / 2) % 4, code % 2
    mag = torch.where(exponent == 0, mantissa / 2, torch.exp2(exponent - 1) * (1 + mantissa / 2))
    where = torch.arange(k, device=codes.device) // 32
    return sign * mag * torch.exp2(scales.double() - 127)[:, where]


def _exact_plan(experts, e):
    flat = experts.reshape(-1).cpu().tolist()
    lists = [[] for _ in range(e)]
    for i, v in enumerate(flat):
        if v >= 0:
            lists[v].append(i)
    order, offsets, rows = [], [0], [-1] * len(flat)
    for members in lists:
        for i in members:
            rows[i] = len(order)
            order.append(i)
        offsets.append(len(order))
    order += [-1] * (len(flat) - len(order))
    make = lambda v: torch.tensor(v, dtype=torch.int32, device=experts.device)  # noqa: E731
    return make(offsets), make(order), make(rows).view_as(experts)


def _exact_route(case, s):
    x = s["logits"].double().requires_grad_(True)
    p = torch.softmax(x, dim=1) if case["scoring"] == "softmax" else torch.sigmoid(x)
    p = torch.where(torch.isneginf(x), torch.zeros_like(p), p)
    with torch.no_grad():
        key = x.detach() if s["bias"] is None else (p + s["bias"].double()).masked_fill(torch.isneginf(x), -math.inf)
        if case["groups"] > 1:
            key = key.masked_fill(~_kept_groups(key, case), -math.inf)
        experts = torch.argsort(-key, dim=1, stable=True)[:, :case["k"]]
        chosen = torch.gather(key, 1, experts) > -math.inf
    score = torch.gather(p, 1, experts) * chosen
    weights = score
    if case["renorm"]:
        total = score.sum(dim=1, keepdim=True)
        weights = score / torch.where(total > 0, total, torch.ones_like(total))
    weights = weights * case["scale"]
    ids = experts.masked_fill(~chosen, -1).to(torch.int32)
    offsets, order, rows = _exact_plan(ids, case["e"])
    out = {"weights": weights.detach(), "experts": ids, "offsets": offsets, "order": order, "rows": rows}
    if case["train"]:
        (grad,) = torch.autograd.grad((weights * s["grad"].double() * chosen).sum(), x)
        out["grad"] = grad.nan_to_num(0.0)          # rows that are -inf throughout have no distribution: no gradient either
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op == "route":
        return _exact_route(case, s)
    if op == "quantize":
        return _exact_quantized(s["x"]) if case["dim"] == 1 else _exact_quantized(s["x"].t()).t()
    if op == "matmul":
        return _exact_quantized(s["x"]) @ _exact_values(s["codes"], s["scales"], case["k"]).t()
    if op == "linear":
        x, w, dy = s["x"], s["w"], s["dy"]
        return {"y": _exact_quantized(x) @ _exact_quantized(w.t()).t(), "dx": _exact_quantized(dy) @ _exact_quantized(w).t(),
                "dw": _exact_quantized(x.t()) @ _exact_quantized(dy.t()).t()}
    offsets, order, rows = _exact_plan(s["experts"], case["e"])
    xq = _exact_quantized(s["x"])
    t, k, d, f = case["t"], case["k"], case["d"], case["f"]
    out = torch.zeros(t * k if op == "up" else t, f if op == "up" else d, dtype=torch.float64, device=xq.device)
    flat_weights = s["weights"].double().flatten()
    for i, (lo, hi) in enumerate(zip(offsets.tolist(), offsets.tolist()[1:])):
        if lo == hi:
            continue
        w = _exact_values(s["codes"][i], s["scales"][i], d if op == "up" else f)
        pairs = order[lo:hi].long()
        if op == "up":
            z = (xq[pairs // k] @ w.t()).unflatten(1, (f, 2))
            out[lo:hi] = torch.nn.functional.silu(z[..., 0]) * z[..., 1]
        else:
            out.index_add_(0, pairs // k, (xq[lo:hi] @ w.t()) * flat_weights[pairs].unsqueeze(1))
    return out
