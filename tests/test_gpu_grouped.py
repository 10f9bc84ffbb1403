"""Products grouped by ragged runs of rows against the definition in 64 bits."""
import ctypes

import pytest
import torch

import blocks_reference as ref
import tritonix
from tritonix_amd import _C
from tritonix_amd.ops import grouped as module

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def weights(device, groups, k, n, dtype, layout, seed):
    if layout == "nn":
        return ref.draw(device, groups, k, n, dtype=dtype, seed=seed, scale=k ** -0.5)
    return ref.draw(device, groups, n, k, dtype=dtype, seed=seed, scale=k ** -0.5).transpose(1, 2)


def step(x, w, offsets, dy):
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    y = tritonix.grouped_matmul(x, w, offsets)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    return {"y": y.detach(), "dx": dx, "dw": dw}


def compare(got, want, dtype):
    for name in got:
        ref.check(name, got[name], want[name], dtype)


def offsets_of(device, counts, first=0):
    out = [first]
    for c in counts:
        out.append(out[-1] + c)
    return torch.tensor(out, dtype=torch.int32, device=device)


# counts of the groups' rows, rows ahead of the first and behind the last
RAGGED = [([1], 0, 0), ([5, 0, 3], 0, 0), ([0, 0, 0], 0, 4), ([64, 64], 0, 0), ([1, 127, 0, 129, 63], 3, 5), ([0, 300, 0, 1], 0, 17), ([2] * 70, 1, 1),
          ([0] * 62 + [3], 0, 0), ([0] * 63 + [9, 1], 2, 0), ([7, 0] * 100, 0, 30), ([1000], 24, 0)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["nn", "nt"])
@pytest.mark.parametrize("case", range(len(RAGGED)))
def test_ragged_groups(device, dtype, layout, case):
    counts, ahead, behind = RAGGED[case]
    k, n = [(64, 128), (100, 70), (72, 264), (33, 50), (130, 8)][case % 5]
    rows = ahead + sum(counts) + behind
    x, w = ref.draw(device, rows, k, dtype=dtype, seed=case), weights(device, len(counts), k, n, dtype, layout, case + 1)
    offsets, dy = offsets_of(device, counts, ahead), ref.draw(device, rows, n, dtype=dtype, seed=case + 2)
    got = step(x, w, offsets, dy)
    compare(got, ref.grouped(x, w, offsets, dy), dtype)
    assert torch.equal(tritonix.grouped_matmul(x, w, offsets.long()), got["y"])
    assert not got["y"][:ahead].any() and not got["y"][rows - behind:].any() and not got["dx"][:ahead].any() and not got["dx"][rows - behind:].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k,n", [(1, 1), (2, 3), (3, 200), (200, 5), (7, 9), (16, 2), (65, 63), (1030, 24), (24, 1030)])
def test_sizes(device, dtype, k, n):
    counts = [3, 0, 70, 1]
    x, w, dy = ref.draw(device, 80, k, dtype=dtype, seed=1), weights(device, 4, k, n, dtype, "nn", 2), ref.draw(device, 80, n, dtype=dtype, seed=3)
    offsets = offsets_of(device, counts, 2)
    compare(step(x, w, offsets, dy), ref.grouped(x, w, offsets, dy), dtype)
    wt = weights(device, 4, k, n, dtype, "nt", 2)
    compare(step(x, wt, offsets, dy), ref.grouped(x, wt, offsets, dy), dtype)


TILES = {torch.bfloat16: [(256, 256), (256, 128), (128, 256), (128, 128), (64, 128), (64, 64), (32, 128), (32, 64)], torch.float32: [(32, 64), (64, 64), (32, 128)]}
TILES[torch.float16] = TILES[torch.bfloat16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tile", range(8))
@pytest.mark.parametrize("aligned", [True, False])
def test_every_tile(device, dtype, tile, aligned, monkeypatch):
    """Each tile over groups shorter and longer than it, of one row and of none, more slabs of k than its ring holds."""
    if tile >= len(TILES[dtype]):
        pytest.skip("not a tile of this type")
    bm, bn = TILES[dtype][tile]
    made = module._args

    def with_tile(form, *args):
        g = made(form, *args)
        g.block_m, g.block_n = bm, bn
        return g

    monkeypatch.setattr(module, "_args", with_tile)
    counts = [bm + 1, 0, 1, 2 * bm, 3, 330]
    k, n = (512, 2 * bn + 64) if aligned else (517, bn + 37)
    ahead, behind = 5, bm + 3
    rows = ahead + sum(counts) + behind
    offsets, dy = offsets_of(device, counts, ahead), ref.draw(device, rows, n, dtype=dtype, seed=3)
    x = ref.draw(device, rows, k, dtype=dtype, seed=1)
    for layout in ("nn", "nt"):
        w = weights(device, len(counts), k, n, dtype, layout, 2)
        want = ref.grouped(x, w, offsets, dy)
        ref.check("y", tritonix.grouped_matmul(x, w, offsets), want["y"], dtype)
    if bm >= 64 or dtype == torch.float32:
        ref.check("dw", module._weight_gradient(x, dy, offsets), want["dw"], dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tile", range(6))
@pytest.mark.parametrize("parts", [2, 3, 7, 40])
def test_k_in_parts(device, dtype, tile, parts, monkeypatch):
    """k, or a group's rows, cut in parts: more of them than a group has slabs, the last one short."""
    tiles = [(128, 128), (64, 128), (64, 64), (32, 128), (32, 64), (64, 64)] if dtype != torch.float32 else TILES[torch.float32] * 2
    made, (bm, bn) = module._args, tiles[tile]

    def with_parts(form, *args):
        g = made(form, *args)
        g.block_m, g.block_n, g.parts = bm, bn, parts
        return g

    monkeypatch.setattr(module, "_args", with_parts)
    counts, ahead, behind = [bm + 1, 0, 1, 3, 530], 5, 9
    rows = ahead + sum(counts) + behind
    offsets = offsets_of(device, counts, ahead)
    for k, n in ((512, bn + 64), (333, bn + 37), (40, 72)):
        x, dy = ref.draw(device, rows, k, dtype=dtype, seed=1), ref.draw(device, rows, n, dtype=dtype, seed=3)
        for layout in ("nn", "nt"):
            w = weights(device, len(counts), k, n, dtype, layout, 2)
            want = ref.grouped(x, w, offsets, dy)
            ref.check(f"y {k} {layout}", module._rows_product(x, w, offsets), want["y"], dtype)
        if bm >= 64 or dtype == torch.float32:
            ref.check(f"dw {k}", module._weight_gradient(x, dy, offsets), want["dw"], dtype)


# counts of the groups' rows, rows ahead and behind, k, n: a row each, runs longer than 8 rows, many groups, short and long k
FEW = [([1], 0, 0, 1, 1), ([0, 3, 0], 0, 0, 7, 5), ([1, 0, 1], 1, 2, 65, 9), ([0, 8], 0, 0, 640, 200), ([2, 0, 9, 1, 0], 3, 2, 1024, 136), ([0, 0, 0, 17, 0, 0, 0], 1, 2, 300, 77),
       ([1, 0] * 60, 0, 3, 520, 600), ([4] * 9, 0, 0, 1030, 70), ([0] * 130 + [25, 3], 9, 40, 72, 40), ([3, 5], 0, 0, 8200, 24), ([1, 2, 0, 8, 4, 5], 2, 1, 9000, 20), ([1, 0, 2], 1, 1, 2100, 210), ([0, 0, 1], 0, 0, 1029, 8), ([3, 1], 0, 4, 1090, 1029),
       ([1, 0] * 60, 0, 3, 2050, 600)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", range(len(FEW)))
@pytest.mark.parametrize("pad,offset", [(0, 0), (64, 64), (1, 3)])
@pytest.mark.parametrize("layout", ["nt", "nn"])
def test_few_rows(device, dtype, case, pad, offset, layout):
    """Few rows, streamed: groups of none to 25 rows, rows of the weights on lines of memory and off them, NaN between them that nothing may read."""
    counts, ahead, behind, k, n = FEW[case]
    rows, groups = ahead + sum(counts) + behind, len(counts)

    def strided(m, columns, pitch, seed, scale=1.0):
        whole = torch.full((offset + m * pitch + 8,), float("nan"), dtype=dtype, device=device)
        out = whole[offset:offset + m * pitch].view(m, pitch)[:, :columns]
        out.copy_(ref.draw(device, m, columns, dtype=dtype, seed=seed, scale=scale))
        return out

    own, inner = (n, k) if layout == "nt" else (k, n)
    pitch = (inner + 63) // 64 * 64 if pad == 64 else inner + pad
    x, flat = strided(rows, k, k + pad, 1), strided(groups * own, inner, pitch, 2, k ** -0.5)
    w = flat.as_strided((groups, k, n), (own * pitch, 1, pitch) if layout == "nt" else (own * pitch, pitch, 1), flat.storage_offset())
    offsets = offsets_of(device, counts, ahead)
    if n > 1 and k > 1:
        g = module._args(_C.GROUPED_ROWS, x, w, None, offsets, n, k, *w.stride())
        used = min(rows, groups)
        words = dtype == torch.float32 or (pitch | k + pad | offset) % 2 == 0 or used * n * k <= 8 << 20
        streamed = (k >= 2048 or used * n <= 16384) and words if layout == "nt" else rows <= 8 and n >= 8 and k >= 1024 and used * ((n + 63) // 64) <= 128
        assert _C.load().tnx_grouped_route(ctypes.byref(g), None) == (2 if streamed else 1)
    y = tritonix.grouped_matmul(x, w, offsets)
    ref.check("y", y, ref.grouped(x, w, offsets)["y"], dtype)
    assert not y[:ahead].any() and not y[rows - behind:].any()
    again = tritonix.grouped_matmul(x, w, offsets)
    assert torch.equal(y, again)
    # a row's numbers are its own
    bad = ahead + sum(counts) - 1
    x[bad] = float("nan")
    got = tritonix.grouped_matmul(x, w, offsets)
    others = torch.arange(rows, device=device) != bad
    assert torch.equal(got[others], y[others]) and got[bad].isnan().all()


def test_bounds_past_32_bits(device):
    """int64 bounds that 32 bits do not hold are the nearest inside, as all that lie outside."""
    x, w = ref.draw(device, 64, 256, seed=1), weights(device, 4, 256, 40, torch.bfloat16, "nn", 2)
    wide = torch.tensor([-2 ** 40, 10, 2 ** 32 + 5, 7, 2 ** 62], device=device)
    y = tritonix.grouped_matmul(x, w, wide)
    ref.check("y", y, ref.grouped(x, w, torch.tensor([0, 10, 64, 64, 64]))["y"], torch.bfloat16)
    leaves = [t.detach().requires_grad_(True) for t in (x, w)]
    got = torch.autograd.grad(tritonix.grouped_matmul(*leaves, wide), leaves, y)
    want = torch.autograd.grad(tritonix.grouped_matmul(*leaves, torch.tensor([0, 10, 64, 64, 64], dtype=torch.int32, device=device)), leaves, y)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("bounds", [[-5, 10, 20, 30], [0, 30, 10, 40], [50, 40, 30, 20], [0, 2 ** 31 - 1, 5, 7], [7, 7, 7, 7], [-(2 ** 31), -1, 0, 0], [40, 40, 40, 99]])
def test_bounds_outside_of_the_rows(device, bounds):
    """Whatever the bounds hold, they are taken into the rows and to a sequence that does not decrease."""
    x, w, dy = ref.draw(device, 40, 64, seed=1), weights(device, 3, 64, 96, torch.bfloat16, "nn", 2), ref.draw(device, 40, 96, seed=3)
    offsets = torch.tensor(bounds, dtype=torch.int32, device=device)
    compare(step(x, w, offsets, dy), ref.grouped(x, w, offsets, dy), torch.bfloat16)
    wide = torch.tensor([v * 2 ** 20 if abs(v) > 40 else v for v in bounds], dtype=torch.int64, device=device)
    compare(step(x, w, wide, dy), ref.grouped(x, w, wide, dy), torch.bfloat16)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(device, dtype):
    offsets = offsets_of(device, [20, 0, 41, 9])
    big, w0, g0 = ref.draw(device, 200, 300, dtype=dtype, seed=1), ref.draw(device, 6, 140, 150, dtype=dtype, seed=2, scale=0.1), ref.draw(device, 200, 300, dtype=dtype, seed=3)
    k, n = 90, 70
    xs = {"pitch": big[:70, 3:3 + k], "every other row": big[:140:2, :k], "columns": big[:k, :70].t(), "every other column": big[:70, :2 * k:2]}
    ws = {"pitch": w0[1:5, 2:2 + k, 1:1 + n], "transposed": w0[:4, :n, :k].transpose(1, 2), "transposed, every other row": w0[:4, :2 * n:2, :k].transpose(1, 2),
          "one for all": w0[:1, :k, :n].expand(4, k, n), "backwards": w0[:4, :k, :n].flip(2)}
    for nx, x in xs.items():
        for nw, w in ws.items():
            dy = g0[:70, 5:5 + n]
            got, want = step(x, w, offsets, dy), ref.grouped(x, w, offsets, dy)
            for name in got:
                ref.check(f"{nx}, {nw}: {name}", got[name], want[name], dtype)


def test_empty_sizes(device):
    offsets = torch.zeros(4, dtype=torch.int32, device=device)
    w = weights(device, 3, 16, 24, torch.bfloat16, "nn", 1)
    got = step(torch.empty(0, 16, dtype=torch.bfloat16, device=device), w, offsets, torch.empty(0, 24, dtype=torch.bfloat16, device=device))
    assert got["y"].shape == (0, 24) and got["dx"].shape == (0, 16) and not got["dw"].any()
    got = step(torch.empty(5, 0, dtype=torch.bfloat16, device=device), w[:, :0], offsets + 5, ref.draw(device, 5, 24))
    assert not got["y"].any() and got["dx"].shape == (5, 0) and got["dw"].shape == (3, 0, 24)


def test_numbers_that_are_none_stay_in_their_rows(device):
    """NaN in a row or in a group's weight shows in that group's rows alone, also through the slab of k that is loaded apart."""
    for k, n in ((128, 128), (100, 70)):
        counts = [30, 50, 1, 40]
        x, w = ref.draw(device, 130, k, seed=1), weights(device, 4, k, n, torch.bfloat16, "nn", 2)
        offsets = offsets_of(device, counts)
        clean = tritonix.grouped_matmul(x, w, offsets)
        x[33] = float("nan")
        x[125] = float("inf")                               # (a row of no group)
        w[3] = float("nan")
        y = tritonix.grouped_matmul(x, w, offsets)
        assert y[33].isnan().all() and y[81:121].isnan().all() and not y[121:].any()
        keep = [i for i in range(81) if i != 33]
        assert torch.equal(y[keep], clean[keep])
        dw = module._weight_gradient(x, clean, offsets)
        assert dw[1].isnan().all() and not dw[0].isnan().any() and not dw[2].isnan().any() and not dw[3].isnan().any()


def test_gradients_against_differences(device):
    h, offsets = 1e-3, offsets_of(device, [4, 0, 7], 1)
    x, w, dy = ref.draw(device, 14, 20, dtype=torch.float32, seed=1), weights(device, 3, 20, 12, torch.float32, "nn", 2), ref.draw(device, 14, 12, dtype=torch.float32, seed=3)
    got, want = step(x, w, offsets, dy), ref.grouped(x, w, offsets, dy)
    for name, t in (("x", x), ("w", w)):
        direction = ref.draw("cpu", *t.shape, dtype=torch.float64, seed=4)
        loss = []
        for sign in (1, -1):
            moved = t.double().cpu() + sign * h * direction
            y = _plain(moved if name == "x" else x.double().cpu(), moved if name == "w" else w.double().cpu(), offsets.tolist())
            loss.append((y * dy.double().cpu()).sum())
        difference = (loss[0] - loss[1]) / (2 * h)           # (exact but for 64-bit rounding: the loss is linear along one operand)
        bound = (want["d" + name][1] * direction.abs()).sum() + 1e-9 * want["d" + name][0].abs().sum()
        assert abs((got["d" + name].double().cpu() * direction).sum() - difference) <= bound, name


def _plain(x, w, bounds):
    y = torch.zeros(x.shape[0], w.shape[2], dtype=torch.float64)
    for g, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
        y[lo:hi] = x[lo:hi] @ w[g]
    return y


def test_from_a_graph_with_other_bounds(device):
    """The bounds are read when the graph runs: a replay takes the groups that they hold then."""
    rows, groups, k, n = 200, 9, 136, 72
    x, w, dy = ref.draw(device, rows, k, seed=1), weights(device, groups, k, n, torch.bfloat16, "nn", 2), ref.draw(device, rows, n, seed=3)
    offsets = torch.linspace(0, rows, groups + 1, device=device).to(torch.int32)
    x.requires_grad_(True), w.requires_grad_(True)

    def once():
        y = tritonix.grouped_matmul(x, w, offsets)
        return [y.detach(), *torch.autograd.grad(y, (x, w), dy)]

    once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = once()
    for i in range(4):
        bounds = torch.randint(0, rows + 1, (groups + 1,), generator=torch.Generator().manual_seed(i)).sort().values
        offsets.copy_(bounds.to(torch.int32))
        want = once()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


def test_a_routed_block_trains(device):
    """norm, router, the experts' two products and the join, as a training program strings them together: every gradient against the same block
    in 64 bits.  Rounded between the operators, so the bound is that of bfloat16 through eight of them: 8 roundings of 2^-8 each, relative to the gradient's norm."""
    t, d, f, e, k = 60, 64, 48, 6, 2
    h0 = ref.draw(device, t, d, seed=1)
    parts = {"h": h0, "gain": 1 + ref.draw(device, d, seed=2, scale=0.1), "shift": ref.draw(device, d, seed=3, scale=0.1),
             "router": ref.draw(device, d, e, seed=4, scale=0.2), "up": ref.draw(device, e, d, 2 * f, seed=5, scale=0.1), "down": ref.draw(device, e, f, d, seed=6, scale=0.1)}
    leaves = {name: v.detach().clone().requires_grad_(True) for name, v in parts.items()}
    x = tritonix.layer_norm(leaves["h"], leaves["gain"], leaves["shift"])
    routing = tritonix.moe_route(tritonix.linear(x, leaves["router"]), k)
    rows = x[torch.div(routing.order, k, rounding_mode="floor").long()]
    both = tritonix.grouped_matmul(rows, leaves["up"], routing.offsets)
    act = torch.nn.functional.silu(both[:, 0::2]) * both[:, 1::2]
    out = tritonix.grouped_matmul(act, leaves["down"], routing.offsets)
    y = leaves["h"] + (out[routing.rows.long()] * routing.weights.unsqueeze(-1).to(out.dtype)).sum(dim=1)
    dy = ref.draw(device, t, d, seed=7)
    grads = torch.autograd.grad(y, list(leaves.values()), dy)

    v = {name: p.double().cpu().requires_grad_(True) for name, p in parts.items()}
    x = torch.nn.functional.layer_norm(v["h"], (d,), v["gain"], v["shift"])
    chosen = routing.experts.cpu().long()
    score = torch.softmax(x @ v["router"], dim=1).gather(1, chosen)
    weight = score / score.sum(dim=1, keepdim=True)
    total = v["h"]
    for j in range(k):
        both = torch.bmm(x.unsqueeze(1), v["up"][chosen[:, j]]).squeeze(1)
        act = torch.nn.functional.silu(both[:, 0::2]) * both[:, 1::2]
        total = total + torch.bmm(act.unsqueeze(1), v["down"][chosen[:, j]]).squeeze(1) * weight[:, j:j + 1]
    want = torch.autograd.grad(total, list(v.values()), dy.double().cpu())
    assert (y.detach().double().cpu() - total.detach()).norm() <= 8 * 2.0 ** -8 * total.detach().norm()
    for name, a, b in zip(parts, grads, want):
        assert (a.double().cpu() - b).norm() <= 8 * 2.0 ** -8 * b.norm(), name


def test_route_of_short_rows(device):
    """Rows shorter than a 16-byte chunk are refused by the entry point and padded by the Python side."""
    x, w, offsets = ref.draw(device, 10, 65), ref.draw(device, 2, 65, 3), offsets_of(device, [5, 5])
    g = module._args(_C.GROUPED_ROWS, x, w, None, offsets, 3, 65, *w.stride())
    lib = _C.load()
    assert lib.tnx_grouped_route(ctypes.byref(g), None) == 0
    y = torch.empty(10, 3, dtype=x.dtype, device=device)
    g.c = y.data_ptr()
    assert lib.tnx_grouped(ctypes.byref(g)) == _C.E_UNSUPPORTED
    ref.check("y", tritonix.grouped_matmul(x, w, offsets), ref.grouped(x, w, offsets)["y"])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("workspace", [False, True])
def test_no_k_through_the_entry_point(device, dtype, workspace):
    """k of 0: every row is the sum of nothing, with a workspace to cut k in and without."""
    rows, n = 70, 40
    y = torch.full((rows, n), float("nan"), dtype=dtype, device=device)
    offsets = torch.tensor([3, 20, 66], dtype=torch.int32, device=device)
    scratch = torch.empty(1 << 16, dtype=torch.uint8, device=device)
    g = _C.GroupedArgs(c=y.data_ptr(), offsets=offsets.data_ptr(), rows=rows, n=n, k=0, stride_ar=0, stride_ak=1, stride_group=0, stride_bk=n, stride_bn=1, groups=2,
                       dtype={torch.float16: _C.F16, torch.bfloat16: _C.BF16, torch.float32: _C.F32}[dtype], stream=torch.cuda.current_stream().cuda_stream)
    if workspace:
        g.workspace, g.workspace_bytes = scratch.data_ptr(), scratch.numel()
    assert _C.load().tnx_grouped(ctypes.byref(g)) == _C.OK
    assert not y.isnan().any() and not y.any()
