"""Definitions in 64 bits for the tests of the microscaled products and of the routing (numpy, on the CPU)."""
import numpy as np
import torch

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantize(x):
    """[rows, k] -> (codes [rows, kp], exponents [rows, kp / 32], values [rows, k]); a block that is not finite throughout has exponent 128 and NaN values."""
    x = np.asarray(x, dtype=np.float64)
    rows, k = x.shape
    kp = -(-k // 32) * 32
    p = np.zeros((rows, kp))
    p[:, :k] = x
    blocks = p.reshape(rows, -1, 32)
    bad = ~np.isfinite(blocks).all(axis=2)
    safe = np.where(bad[..., None], 0.0, blocks)
    top = np.abs(safe).max(axis=2)
    mant, ex = np.frexp(top)                              # top = mant * 2^ex, 0.5 <= mant < 1
    e = np.clip(np.where(top > 0, ex - 1, -10000) - 2, -127, 127)
    v = np.abs(safe) / np.exp2(e)[..., None]
    # nearest level, ties to the even code
    dist = np.abs(v[..., None] - LEVELS)
    best = dist.min(axis=-1, keepdims=True)
    tied = dist == best
    order = np.where(np.arange(8) % 2 == 0, np.arange(8), np.arange(8) + 100)
    code = np.where(tied, order, 1000).argmin(axis=-1)
    value = np.sign(safe) * LEVELS[code] * np.exp2(e)[..., None]
    value[bad] = np.nan
    code = code + 8 * np.signbit(safe)
    code[bad] = 0
    return code.reshape(rows, kp), np.where(bad, 128, e), value.reshape(rows, kp)[:, :k]


def values(x, dim=-1):
    """What a float tensor (any device) quantised along ``dim`` stands for, float64."""
    a = x.detach().cpu().double().numpy()
    if a.ndim == 3:
        return np.stack([values(torch.from_numpy(m), dim) for m in a])
    return quantize(a)[2] if dim in (-1, 1) else quantize(a.T)[2].T


def product_bound(a, b, k):
    """How far 32-bit sums may be from a @ b: every one of k / 32 additions of a block's sum, and a block's own, is off by a unit in the last place
    of what has been summed at most (truncation allowed)."""
    return 2.0 ** -23 * (k / 32 + 8) * (np.abs(a) @ np.abs(b))


def rounding(ref, dtype):
    """Half a unit in the last place of a result: 2^(exponent - significant bits), or half the smallest subnormal."""
    bits, smallest = {torch.bfloat16: (8, 2.0 ** -133), torch.float16: (11, 2.0 ** -24), torch.float32: (24, 2.0 ** -149)}[dtype]
    return np.maximum(np.exp2(np.floor(np.log2(np.maximum(np.abs(ref), 2.0 ** -200))) - bits), smallest / 2)


def activation(g, name):
    if name == "silu":
        return g / (1 + np.exp(-g))
    return 1 / (1 + np.exp(-g)) if name == "sigmoid" else g


def gated(z, dz, name):
    """Gated columns of z (gate even) and a bound on their error where z is off by dz: silu's and the sigmoid's slopes are below 1.1; the gate itself is good to 2^-20."""
    g, l, dg, dl = z[:, 0::2], z[:, 1::2], dz[:, 0::2], dz[:, 1::2]
    act = activation(g, name)
    return act * l, 1.1 * dg * (np.abs(l) + dl) + np.abs(act) * dl + 2.0 ** -20 * np.abs(act * l)


def plan(experts, num_experts):
    flat = experts.reshape(-1).tolist()
    order, offsets, rows = [], [0], [-1] * len(flat)
    for e in range(num_experts):
        for i, v in enumerate(flat):
            if v == e:
                rows[i] = len(order)
                order.append(i)
        offsets.append(len(order))
    order += [-1] * (len(flat) - len(order))
    return offsets, order, rows


def route(logits, k, scoring="softmax", bias=None, num_groups=1, top_groups=1, group_top=1, renormalize=True, scale=1.0):
    """Row by row, from the definition: (weights, experts)."""
    x = logits.detach().cpu().double().numpy()
    b = None if bias is None else bias.cpu().double().numpy()
    tokens, n = x.shape
    weights, experts = np.zeros((tokens, k)), np.full((tokens, k), -1)
    for t in range(tokens):
        row = x[t]
        if np.isnan(row).any() or (scoring == "softmax" and (row == np.inf).any()):
            weights[t] = np.nan
            continue
        if (row == -np.inf).all():
            continue
        if scoring == "softmax":
            s = np.exp(row - row.max())
            s /= s.sum()
        else:
            with np.errstate(over="ignore"):
                s = 1 / (1 + np.exp(-row))
        key = row.copy() if b is None else np.where(row == -np.inf, -np.inf, s + b)
        key[np.isnan(key)] = -np.inf
        if num_groups > 1:
            size = n // num_groups
            worth = []
            for g in range(num_groups):
                best = sorted(key[g * size:(g + 1) * size], reverse=True)[:group_top]
                best = [v for v in best if v > -np.inf]
                worth.append(sum(best) if best else -np.inf)
            keep = sorted(range(num_groups), key=lambda g: (-worth[g], g))[:top_groups]
            for g in range(num_groups):
                if g not in keep:
                    key[g * size:(g + 1) * size] = -np.inf
        chosen = [e for e in sorted(range(n), key=lambda e: (-key[e], e)) if key[e] > -np.inf][:k]
        total = sum(s[e] for e in chosen)
        for j, e in enumerate(chosen):
            experts[t, j] = e
            weights[t, j] = scale * s[e] / (total if renormalize and total > 0 else 1.0)
            if renormalize and total == 0:
                weights[t, j] = 0.0
    return weights, experts
