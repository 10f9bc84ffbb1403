"""Mixture of experts: routing of tokens, and the routed, gated feed-forward block on microscaled 4-bit weights.

    routing = moe_route(logits, top_k)                  # who goes where, with which weight
    y = moe_ffn(x, w12, w3, routing)                    # sum over a token's experts of weight * swiglu_ffn(x, w12[e], w3[e])

``moe_ffn`` is ``moe_glu`` (the experts' gated up-projections, rows sorted by expert) and ``moe_down`` (their down-projections,
joined per token).  ``w12[e, d, 2f]`` is interleaved column-wise like ``glu``'s; both weights are ``MXTensor`` batches quantised along the dimension
that is summed over (``mx_quantize(w, dim=-2)`` or ``MXTensor.from_codes(..., dim=-2)``).  Nothing here waits for the GPU: the
rows of each expert are counted and found on it.

The router is trained through ``Routing.weights``, which carries its gradient; the experts' products are for answering and pass none, neither to x nor
to the routing's weights: where one of those asks for its gradient, differentiating their result is an error.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from tritonix_amd import _C
from tritonix_amd.ops import mx as _mx
from tritonix_amd.ops.mx import MXTensor, dtype_code, epilogue_of, gemm_args, launch, on_device, operand, raise_for_status, takes_rows, underived
from tritonix_amd.kernel import _stream_of

__all__ = ["Routing", "moe_route", "moe_route_backward", "moe_plan", "moe_glu", "moe_down", "moe_ffn"]

_SCORING = {"softmax": 0, "sigmoid": 1}


@dataclass
class Routing:
    """Where each token goes.

    ``weights[t, k]`` (float32) and ``experts[t, k]`` (int32, -1: an empty slot) per token; ``order[t * k]``: the pairs token * k + slot sorted
    by expert, by pair within one, then -1; expert e has ``order[offsets[e]:offsets[e + 1]]``; ``rows[t, k]``: each pair's place in ``order`` (-1: none)."""
    weights: torch.Tensor
    experts: torch.Tensor
    offsets: torch.Tensor
    order: torch.Tensor
    rows: torch.Tensor
    num_experts: int
    scoring: Optional[str] = "softmax"         # None: the choice was made elsewhere (moe_plan), its scores are not known
    renormalize: bool = True
    scale: float = 1.0

    @property
    def tokens(self) -> int:
        return self.experts.shape[0]

    @property
    def top_k(self) -> int:
        return self.experts.shape[1]


def _scratch(args, tokens: int, top_k: int, num_experts: int, device) -> Optional[torch.Tensor]:
    nbytes = int(_C.load().tnx_moe_workspace_bytes(tokens, top_k, num_experts))
    if not nbytes:
        return None
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    args.workspace, args.workspace_bytes = ws.data_ptr(), nbytes
    return ws


def _plan_buffers(args, tokens: int, top_k: int, num_experts: int, device):
    pairs = tokens * top_k
    offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=device)
    order = torch.empty(pairs, dtype=torch.int32, device=device)
    rows = torch.empty((tokens, top_k), dtype=torch.int32, device=device)
    args.offsets, args.order, args.rows = offsets.data_ptr(), order.data_ptr(), rows.data_ptr()
    args.tokens, args.top_k, args.num_experts = tokens, top_k, num_experts
    return offsets, order, rows


def _check_counts(name: str, top_k: int, num_experts: int) -> None:
    if not 1 <= num_experts <= _C.MOE_MAX_EXPERTS:
        raise ValueError(f"{name}: {num_experts} experts (1 to {_C.MOE_MAX_EXPERTS} are built)")
    if not 1 <= top_k <= _C.MOE_MAX_TOP_K:
        raise ValueError(f"{name}: top_k {top_k} (1 to {_C.MOE_MAX_TOP_K} are built)")


def moe_plan(experts: torch.Tensor, weights: torch.Tensor, num_experts: int) -> Routing:
    """The plan for a choice made elsewhere: ``experts[t, k]`` (int32 or int64; numbers outside ``[0, num_experts)`` are empty
    slots) and ``weights[t, k]``."""
    if experts.dim() != 2 or tuple(weights.shape) != tuple(experts.shape):
        raise ValueError(f"moe_plan expects experts[t,k] and weights[t,k], got {tuple(experts.shape)} and {tuple(weights.shape)}")
    if experts.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"moe_plan: experts are int32 or int64, got {experts.dtype}")
    tokens, top_k = experts.shape
    _check_counts("moe_plan", top_k, num_experts)
    index = on_device("moe_plan", experts, weights)
    if experts.dtype == torch.int64:                       # (numbers past 32 bits are empty slots too)
        experts = torch.where((experts >= 0) & (experts < num_experts), experts, -1)
    experts = experts.to(torch.int32).contiguous()
    weights = weights.to(torch.float32).contiguous()
    a = _C.MoeArgs()
    offsets, order, rows = _plan_buffers(a, tokens, top_k, num_experts, experts.device)
    a.experts = experts.data_ptr()
    ws = _scratch(a, tokens, top_k, num_experts, experts.device)
    launch("moe_plan", index, _C.load().tnx_moe_plan, a)
    del ws
    return Routing(weights, experts, offsets, order, rows, num_experts, scoring=None)


def _route_args(logits: torch.Tensor, bias: Optional[torch.Tensor], top_k: int, options) -> _C.MoeArgs:
    scoring, num_groups, top_groups, group_top, renormalize, scale = options
    a = _C.MoeArgs()
    a.logits, a.bias = logits.data_ptr(), bias.data_ptr() if bias is not None else None
    a.tokens, a.stride_logits = logits.shape[0], logits.stride(0)
    a.num_experts, a.top_k, a.dtype, a.scoring = logits.shape[1], top_k, dtype_code("moe_route", logits.dtype), _SCORING[scoring]
    a.num_groups, a.top_groups, a.group_top, a.renormalize, a.scale = num_groups, top_groups, group_top, int(renormalize), scale
    return a


def _route(logits, bias, top_k, options):
    index = logits.get_device()
    tokens, num_experts = logits.shape
    a = _route_args(logits, bias, top_k, options)
    device = logits.device
    weights = torch.empty((tokens, top_k), dtype=torch.float32, device=device)
    experts = torch.empty((tokens, top_k), dtype=torch.int32, device=device)
    a.weights, a.experts = weights.data_ptr(), experts.data_ptr()
    offsets, order, rows = _plan_buffers(a, tokens, top_k, num_experts, device)
    ws = _scratch(a, tokens, top_k, num_experts, device)
    launch("moe_route", index, _C.load().tnx_moe_route, a)
    del ws
    return weights, experts, offsets, order, rows


class _Route(torch.autograd.Function):
    """What the native side has not taken."""

    @staticmethod
    def forward(ctx, logits, bias, top_k, options):
        out = _route(logits, bias, top_k, options)
        ctx.save_for_backward(logits, out[0], out[1])
        ctx.options = options
        ctx.mark_non_differentiable(*out[1:])
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad, *_):
        logits, weights, experts = ctx.saved_tensors
        return _backward(grad, logits, weights, experts, ctx.options), None, None, None


def moe_route(logits: torch.Tensor, top_k: int, scoring: str = "softmax", bias: Optional[torch.Tensor] = None, num_groups: int = 1,
              top_groups: int = 1, group_top: int = 1, renormalize: bool = True, scale: float = 1.0) -> Routing:
    """Choose ``top_k`` experts for each row of ``logits[t, e]`` (float16, bfloat16 or float32).

    Scores are ``softmax`` or ``sigmoid`` of the logits.  With ``bias[e]`` (float32; a term that balances the load) experts
    rank by score + bias, without by their logit; the bias never enters a weight.  With ``num_groups`` > 1 the experts come in that
    many equal groups and only the ``top_groups`` best may be chosen from, a group being worth the sum of its ``group_top`` (1 or 2; 2 needs a
    bias, since only biased scores are summed) largest keys.  Equal keys: the lower expert.  Weights are the chosen scores, divided by their sum if
    ``renormalize``, times ``scale``.

    A logit of -inf cannot be chosen; slots that nothing is left for hold expert -1 and weight 0 (a row of -inf throughout: all of
    them).  A row with a NaN (softmax: or +inf) gets experts -1 and NaN weights.  ``weights`` carries a gradient if ``logits`` does; the choice is held fixed."""
    if logits.dim() != 2:
        raise ValueError(f"moe_route expects logits[t,e], got {tuple(logits.shape)}")
    renormalize, scale = bool(renormalize), float(scale)
    number = _SCORING.get(scoring)
    if number is not None and (group_top == 1 or bias is not None):
        out = (_mx.native or _mx.find_native()).moe_route(logits, bias, top_k, number, num_groups, top_groups, group_top, renormalize, scale)
        if out is not None:
            return Routing(*out, logits.shape[1], scoring, renormalize, scale)
    tokens, num_experts = logits.shape
    _check_counts("moe_route", top_k, num_experts)
    if top_k > num_experts:
        raise ValueError(f"moe_route: top_k {top_k} of {num_experts} experts")
    if scoring not in _SCORING:
        raise ValueError(f"moe_route: scoring is 'softmax' or 'sigmoid', got {scoring!r}")
    if not 1 <= num_groups <= _C.MOE_MAX_GROUPS or num_experts % num_groups or not 1 <= top_groups <= num_groups:
        raise ValueError(f"moe_route: {top_groups} of {num_groups} groups of {num_experts} experts")
    if group_top not in (1, 2) or (group_top == 2 and bias is None):
        raise ValueError("moe_route: group_top is 1, or 2 with a bias")
    if bias is not None and (tuple(bias.shape) != (num_experts,) or bias.dtype != torch.float32):
        raise ValueError(f"moe_route: bias is float32 [{num_experts}], got {bias.dtype} {tuple(bias.shape)}")
    dtype_code("moe_route", logits.dtype)
    on_device("moe_route", logits, bias)
    if logits.stride(1) != 1 and num_experts > 1:
        logits = logits.contiguous()
    if bias is not None:
        bias = bias.detach().contiguous()
    options = (scoring, num_groups, top_groups, group_top, renormalize, scale)
    if logits.requires_grad and torch.is_grad_enabled():
        out = _Route.apply(logits, bias, top_k, options)
    else:
        out = _route(logits, bias, top_k, options)
    return Routing(*out, num_experts, scoring, renormalize, scale)


def _backward(grad, logits, weights, experts, options):
    out = (_mx.native or _mx.find_native()).moe_backward(grad, logits, weights, experts, _SCORING[options[0]], options[4], options[5])
    if out is not None:
        return out
    _check_field("moe_route_backward", "weights", weights, torch.float32, tuple(grad.shape))
    _check_field("moe_route_backward", "experts", experts, torch.int32, tuple(grad.shape))
    index = on_device("moe_route_backward", grad, logits, weights, experts)
    a = _route_args(logits, None, experts.shape[1], options)
    out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    grad = grad.to(torch.float32).contiguous()
    a.weights, a.experts, a.grad, a.grad_logits = weights.data_ptr(), experts.data_ptr(), grad.data_ptr(), out.data_ptr()
    launch("moe_route_backward", index, _C.load().tnx_moe_route_backward, a)
    return out


def moe_route_backward(grad_weights: torch.Tensor, logits: torch.Tensor, routing: Routing) -> torch.Tensor:
    """Gradient of the logits from that of ``routing.weights``, for the ``routing`` that ``moe_route`` made of these logits."""
    if routing.scoring not in _SCORING:
        raise ValueError("moe_route_backward: the routing of moe_plan has weights from elsewhere, whose gradient of logits is not known")
    if tuple(grad_weights.shape) != (routing.tokens, routing.top_k) or logits.dim() != 2 or tuple(logits.shape) != (routing.tokens, routing.num_experts):
        raise ValueError(f"moe_route_backward: gradient {tuple(grad_weights.shape)} and logits {tuple(logits.shape)} are not of this routing "
                         f"({routing.tokens} tokens, {routing.top_k} of {routing.num_experts} experts)")
    dtype_code("moe_route_backward", logits.dtype)
    if logits.stride(1) != 1 and routing.num_experts > 1:
        logits = logits.contiguous()
    return _backward(grad_weights, logits, routing.weights, routing.experts, (routing.scoring, 1, 1, 1, routing.renormalize, routing.scale))


def _check_field(name: str, field: str, t: torch.Tensor, dtype, shape) -> None:
    """The kernels read a routing as it was made: one that was changed since has to have kept its types and sizes."""
    if t.dtype != dtype or tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{name}: routing.{field} is contiguous {dtype} {shape}, got {t.dtype} {tuple(t.shape)}")


def _check_experts(name: str, x, w, routing: Routing, rows: int) -> None:
    slots = tuple(routing.experts.shape)
    _check_field(name, "offsets", routing.offsets, torch.int32, (routing.num_experts + 1,))
    _check_field(name, "order", routing.order, torch.int32, (routing.tokens * routing.top_k,))
    _check_field(name, "rows", routing.rows, torch.int32, slots)
    _check_field(name, "weights", routing.weights, torch.float32, slots)
    if not isinstance(w, MXTensor) or w.batch is None:
        raise ValueError(f"{name}: the experts' weights are an MXTensor of shape [experts, k, n]")
    if w.batch != routing.num_experts:
        raise ValueError(f"{name}: weights of {w.batch} experts, a routing to {routing.num_experts}")
    if w.dim != -2:
        raise ValueError(f"{name}: weights of shape {w.shape} have to be quantised along the dimension that is summed over (dim=-2)")
    if len(x.shape) != 2 or x.shape[1] != w.k or x.shape[0] != rows:
        raise ValueError(f"{name} expects [{rows}, {w.k}] rows, got {tuple(x.shape)}")


def _grouped(name: str, x, w: MXTensor, routing: Routing, out: torch.Tensor, gather: bool, epilogue: int, index: int) -> None:
    g = gemm_args(x, w, out, epilogue)
    g.experts, g.offsets, g.top_k = routing.num_experts, routing.offsets.data_ptr(), routing.top_k
    if gather:
        g.order = routing.order.data_ptr()
    launch(name, index, _C.load().tnx_mx_gemm, g)


def moe_glu(x, w12: MXTensor, routing: Routing, activation: str = "silu", out_dtype=None) -> torch.Tensor:
    """Gated up-projections of each token's experts: row r of the result, ``[t * k, f]``, belongs to the pair ``routing.order[r]``; rows
    of empty slots come last and are zero.  ``x[t, d]`` is a torch tensor or an ``MXTensor``, ``w12`` an ``MXTensor`` ``[e, d, 2f]``."""
    if out_dtype is None and type(w12) is MXTensor and w12.batch == routing.num_experts and w12.dim == -2 and x.shape[:1] == (routing.tokens,):
        out = (_mx.native or _mx.find_native()).mx_product(x, w12.buffer, w12.code_bytes, w12.rows, w12.k, epilogue_of(activation), routing.num_experts,
                                                           routing.top_k, routing.offsets, routing.order, None, None)
        if out is not None:
            return underived("moe_glu", out, x) if x.requires_grad else out
    _check_experts("moe_glu", x, w12, routing, routing.tokens)
    if w12.rows % 2:
        raise ValueError("the interleaved weight must have an even number of columns")
    if out_dtype is None:
        out_dtype = torch.bfloat16 if isinstance(x, MXTensor) else x.dtype
    dtype_code("moe_glu", out_dtype)
    index = on_device("moe_glu", x, w12, routing.offsets, routing.order)
    xq = x if takes_rows(x) else operand("moe_glu", "x", x, -1)
    out = torch.empty((routing.tokens * routing.top_k, w12.rows // 2), dtype=out_dtype, device=w12.device)
    _grouped("moe_glu", xq, w12, routing, out, True, epilogue_of(activation), index)
    return underived("moe_glu", out, x)


def moe_down(h, w3: MXTensor, routing: Routing, out_dtype=None) -> torch.Tensor:
    """Down-projections of the rows that ``moe_glu`` made, joined: ``out[t] = sum_j weights[t, j] * (h[rows[t, j]] @ w3[e])``, ``[t, d]``.
    Empty slots are left out; where their weight is NaN (``moe_route`` of a row with a NaN) the token's output is NaN.

    The join sums in 32 bits, and so are the products it sums, but for bfloat16 results whose products would take more than 32 MiB: those are rounded to
    bfloat16 first (they are k times the result's size, and writing and reading them is what the join costs), which with eight experts takes the
    error relative to the exact sum from 0.0017 to 0.0024.  ``out_dtype=torch.float32`` keeps them in 32 bits at every size."""
    if out_dtype is None and type(w3) is MXTensor and w3.batch == routing.num_experts and w3.dim == -2:
        out = (_mx.native or _mx.find_native()).mx_product(h, w3.buffer, w3.code_bytes, w3.rows, w3.k, _C.EPI_NONE, routing.num_experts, routing.top_k,
                                                           routing.offsets, None, routing.rows, routing.weights)
        if out is not None:
            return underived("moe_down", out, h, routing.weights) if h.requires_grad or routing.weights.requires_grad else out
    _check_experts("moe_down", h, w3, routing, routing.tokens * routing.top_k)
    if out_dtype is None:
        out_dtype = torch.bfloat16 if isinstance(h, MXTensor) else h.dtype
    code = dtype_code("moe_down", out_dtype)
    index = on_device("moe_down", h, w3, routing.offsets, routing.rows, routing.weights)
    hq = h if takes_rows(h) else operand("moe_down", "h", h, -1)
    n = w3.rows
    rows = routing.tokens * routing.top_k
    in_32_bits = out_dtype != torch.bfloat16 or rows * n * 4 <= _mx.JOIN_BYTES
    y = torch.empty((rows, n), dtype=torch.float32 if in_32_bits else out_dtype, device=w3.device)
    _grouped("moe_down", hq, w3, routing, y, False, _C.EPI_NONE, index)
    out = torch.empty((routing.tokens, n), dtype=out_dtype, device=w3.device)
    with torch.cuda.device(index):
        status = _C.load().tnx_moe_combine(y.data_ptr(), routing.rows.data_ptr(), routing.weights.data_ptr(), out.data_ptr(), routing.tokens,
                                           routing.top_k, n, dtype_code("moe_down", y.dtype), code, _stream_of(index))
    raise_for_status(status, "moe_down")
    return underived("moe_down", out, h, routing.weights)


def moe_ffn(x, w12: MXTensor, w3: MXTensor, routing: Routing, activation: str = "silu", out_dtype=None) -> torch.Tensor:
    """The routed feed-forward block: ``sum over j of weights[t, j] * (act(x W1_e) * (x W2_e)) W3_e`` with e the token's j-th expert."""
    if not isinstance(w3, MXTensor) or not isinstance(w12, MXTensor) or w3.k != w12.rows // 2:
        raise ValueError("moe_ffn expects MXTensor weights w12[e, d, 2f] and w3[e, f, d']")
    return moe_down(moe_glu(x, w12, routing, activation, out_dtype), w3, routing, out_dtype)
