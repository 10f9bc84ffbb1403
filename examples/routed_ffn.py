"""A routed feed-forward block on 4-bit weights: a step that trains the router, a prompt, and single tokens from a HIP graph.

    python -m examples.routed_ffn [tokens] [width] [inner] [experts] [top_k]

The experts' weights are microscaled once (``mx_quantize``; a checkpoint's codes come in through ``MXTensor.from_codes``).  The router is an
``mx_linear`` layer: its product and both gradients' are microscaled too, and the routing's weights carry the gradient to it.
"""
import sys

import torch

import tritonix


def block(x, w_router, w12, w3, top_k):
    logits = tritonix.mx_linear(x, w_router)
    routing = tritonix.moe_route(logits.float(), top_k)
    return tritonix.moe_ffn(x, w12, w3, routing), routing


def main(tokens=2048, width=2048, inner=1024, experts=32, top_k=4, device="cuda"):
    g = torch.Generator("cpu").manual_seed(0)

    def rand(*shape, scale=1.0):
        return (torch.randn(shape, generator=g) * scale).bfloat16().to(device)

    x = rand(tokens, width)
    w_router = rand(width, experts, scale=width ** -0.5)
    w12 = tritonix.mx_quantize(rand(experts, width, 2 * inner, scale=width ** -0.5), dim=-2)
    w3 = tritonix.mx_quantize(rand(experts, inner, width, scale=inner ** -0.5), dim=-2)

    # a step of the router, towards an even load
    w_router.requires_grad_(True)
    _, routing = block(x, w_router, w12, w3, top_k)
    load = torch.zeros(experts, device=device).index_add(0, routing.experts.flatten().long(), routing.weights.flatten())
    before = ((load / tokens - 1.0 / experts) ** 2).sum()
    before.backward()
    with torch.no_grad():
        w_router -= 100.0 * w_router.grad.to(w_router.dtype)

    # answers: a prompt, then one token at a time
    with torch.no_grad():
        y, routing = block(x, w_router, w12, w3, top_k)
        counts = (routing.offsets[1:] - routing.offsets[:-1]).tolist()
        token = x[:1].clone()
        block(token, w_router, w12, w3, top_k)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, _ = block(token, w_router, w12, w3, top_k)
        worst = 0.0
        for t in range(min(4, tokens)):
            token.copy_(x[t:t + 1])
            graph.replay()
            worst = max(worst, float((out - y[t:t + 1]).float().abs().max()))
    print(f"{tokens} tokens, {experts} experts, {top_k} each: rows per expert {min(counts)} to {max(counts)}, uneven load {float(before.detach()):.2e}; "
          f"single tokens differ from the prompt's by {worst:.1e} at most (largest value {float(y.float().abs().max()):.2f})")
    return worst, float(y.float().abs().max())


if __name__ == "__main__":
    main(*(int(v) for v in sys.argv[1:]))
