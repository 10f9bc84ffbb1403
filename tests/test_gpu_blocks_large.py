"""Linear layers, layer normalisation and grouped products whose elements are past 32 bits, of very many rows, and from several threads at once."""
import importlib
import threading

import pytest
import torch

import blocks_reference as ref
import tritonix

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
ROWS, WIDE = 70000, 32768                  # 2.3e9 elements: offsets of the last 4485 rows do not fit 31 bits


def random(device, *shape, scale=1.0, seed=0):
    return torch.empty(shape, dtype=BF16, device=device).normal_(0.0, scale, generator=torch.Generator(device).manual_seed(seed))


LAST = slice(ROWS - 3, ROWS)


def test_a_linear_layer_past_32_bits(device):
    k = 64
    x, w, bias, residual = random(device, ROWS, k), random(device, k, WIDE, scale=0.1, seed=1), random(device, WIDE, seed=2), random(device, ROWS, WIDE, seed=3)
    leaves = [t.requires_grad_(True) for t in (x, w, bias)]
    y = tritonix.linear(x, w, bias, "silu", residual)
    dx, dw, dbias = torch.autograd.grad(y, leaves, residual)
    want = ref.linear(x[LAST], w, bias, "silu", residual[LAST], residual[LAST])
    ref.check("y", y[LAST], want["y"], BF16)
    ref.check("dx", dx[LAST], want["dx"], BF16)
    cols = slice(WIDE - 2, WIDE)                          # (of the sums over the rows the last columns)
    want = ref.linear(x, w[:, cols], bias[cols], "silu", None, residual[:, cols])
    ref.check("dw", dw[:, cols], want["dw"], BF16)
    ref.check("dbias", dbias[cols], want["dbias"], BF16)


def test_few_rows_by_a_weight_past_32_bits(device):
    """A weight of 2.3e9 elements, k-contiguous: its last rows."""
    x, w = random(device, 2, WIDE), random(device, ROWS, WIDE, scale=WIDE ** -0.5, seed=1).t()
    ref.check("y", tritonix.linear(x, w)[:, LAST], ref.linear(x, w[:, LAST])["y"], BF16)


def test_normalisation_past_32_bits(device):
    x, dy, weight, bias = random(device, ROWS, WIDE), random(device, ROWS, WIDE, seed=1), random(device, WIDE, seed=2), random(device, WIDE, seed=3)
    leaves = [t.requires_grad_(True) for t in (x, weight, bias)]
    y = tritonix.layer_norm(x, weight, bias)
    dx, _, dbias = torch.autograd.grad(y, leaves, dy)
    want = ref.layer_norm(x[LAST], weight, bias, 1e-5, dy[LAST])
    ref.check("y", y[LAST], want["y"], BF16)
    ref.check("dx", dx[LAST], want["dx"], BF16)
    column = dy[:, -1].double()
    bound = (ROWS + 2) * ref.E * column.abs().sum() + ref.rounding(column.sum(), BF16)
    assert (dbias[-1].double() - column.sum()).abs() <= bound


def test_more_rows_than_a_launch_has_threads_for(device):
    """70 million short rows, a wave's worth of threads to each."""
    rows, n = 70000000, 8
    x, weight, dy = random(device, rows, n), random(device, n, seed=1), random(device, rows, n, seed=2)
    leaves = [t.requires_grad_(True) for t in (x, weight)]
    y = tritonix.layer_norm(x, weight)
    dx, _ = torch.autograd.grad(y, leaves, dy)
    for first in (0, (1 << 24) - 20, (1 << 26) - 70, rows - 50):        # (around the ends of launches, and the last)
        part = slice(first, first + 50)
        want = ref.layer_norm(x[part], weight, None, 1e-5, dy[part])
        ref.check("y", y[part], want["y"], BF16)
        ref.check("dx", dx[part], want["dx"], BF16)


def test_a_grouped_product_past_32_bits(device):
    """Rows past 32 bits, and of the weights and their gradient."""
    k = 64
    x, w = random(device, ROWS, k), random(device, 3, k, WIDE, scale=0.1, seed=1)
    offsets = torch.tensor([1, 40000, 69000, ROWS - 1], dtype=torch.int32, device=device)
    y = tritonix.grouped_matmul(x, w, offsets)
    part = slice(ROWS - 4, ROWS - 1)
    ref.check("y", y[part], ref.linear(x[part], w[2])["y"], BF16)
    assert not y[0].any() and not y[ROWS - 1].any()
    del x, w, y
    groups, k, n = 128, 4608, 4096                        # 2.4e9 elements of weights
    x, w, dy = random(device, 300, k), random(device, groups, k, n, scale=k ** -0.5, seed=1), random(device, 300, n, seed=2)
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    offsets = torch.tensor([min(300, 2 * g + max(0, 3 * (g - 120))) for g in range(groups + 1)], dtype=torch.int32, device=device)
    y = tritonix.grouped_matmul(x, w, offsets)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    for g in (0, groups - 1):
        rows = slice(int(offsets[g]), int(offsets[g + 1]))
        want = ref.linear(x[rows], w[g], dy=dy[rows])
        ref.check("y", y[rows], want["y"], BF16)
        ref.check("dx", dx[rows], want["dx"], BF16)
        ref.check("dw", dw[g], want["dw"], BF16)


def test_sums_of_more_rows_than_a_grid_has_blocks(device):
    """4.5 million rows: the gradient's pass takes longer blocks of them.  Whole numbers, whose sums are exact."""
    m, n = 4500001, 16
    x, w = random(device, m, 16), random(device, 16, n, seed=1)
    bias = torch.zeros(n, device=device, requires_grad=True)
    dy = torch.randint(-1, 2, (m, n), device=device, generator=torch.Generator(device).manual_seed(1)).to(BF16)
    (got,) = torch.autograd.grad(tritonix.linear(x, w, bias), (bias,), dy)
    assert torch.equal(got.double(), dy.sum(dim=0, dtype=torch.float64))


def test_one_weight_for_all_groups(device):
    """An expanded weight, its groups in the same memory: the gradient sums over them."""
    x, dy = random(device, 200, 72), random(device, 200, 40, seed=1)
    one = random(device, 72, 40, scale=0.1, seed=2).requires_grad_(True)
    offsets = torch.tensor([0, 90, 90, 200], dtype=torch.int32, device=device)
    y = tritonix.grouped_matmul(x, one.expand(3, 72, 40), offsets)
    want = ref.linear(x, one, dy=dy)
    ref.check("y", y.detach(), want["y"], BF16)
    (dw,) = torch.autograd.grad(y, (one,), dy)
    # (each group's gradient is rounded, and their sum)
    parts = [x[a:b].double().t() @ dy[a:b].double() for a, b in ((0, 90), (90, 200))]
    bound = want["dw"][1] + sum(ref.rounding(p, BF16) for p in parts).cpu() * (1 + ref.unit(BF16))
    ref.check("dw", dw, (want["dw"][0], bound), BF16)


def test_threads_on_streams_of_their_own(device):
    """Calls from four threads, each on a stream, with products that are cut along k into growing workspaces: the bits of a single thread's."""
    sizes = [(40, 1000, 2304), (24, 520, 4096), (64, 2000, 2048), (3, 300, 5000)]
    data = []
    for i, (m, n, k) in enumerate(sizes):
        x, w, b = random(device, m, k), random(device, k, n, scale=k ** -0.5, seed=1), random(device, n, seed=2)
        groups = torch.tensor([0, m // 3, m], dtype=torch.int32, device=device)
        data.append((x, w, b, groups, torch.stack([w, w])))

    def work(i):
        x, w, b, groups, pair = data[i]
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y = tritonix.layer_norm(tritonix.linear(leaves[0], leaves[1], leaves[2], "gelu"))
        return [y.detach(), tritonix.grouped_matmul(x, pair, groups), *torch.autograd.grad(y, leaves, y.detach())]

    want = [work(i) for i in range(len(sizes))]
    torch.cuda.synchronize()
    failures = []

    def thread(first):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for turn in range(12):
                    i = (first + turn) % len(sizes)
                    got = work(i)
                    stream.synchronize()
                    if not all(torch.equal(a, c) for a, c in zip(got, want[i])):
                        failures.append((first, turn))
        except Exception as e:  # noqa: BLE001
            failures.append(e)

    threads = [threading.Thread(target=thread, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures


def test_sums_of_more_columns_than_a_launch_has_threads_for(device):
    """The second launches of bias' and parameters' gradients, 16 threads to a column: past 2^28 columns of a linear layer, 2^27 of a normalisation."""
    module = importlib.import_module("tritonix_amd.ops.linear")
    m, n = 65, (1 << 28) + 200
    dy = torch.ones(m, n, dtype=BF16, device=device)
    odd = torch.tensor([0, 5, n // 2, (1 << 28) - 1, 1 << 28, n - 1], device=device)
    dy[m - 1, odd] = 7.0
    dbias = module._gradient(dy, None, 0, False, torch.float32)[1]
    del dy
    want = torch.full((n,), 65.0, device=device)
    want[odd] = 71.0
    assert torch.equal(dbias, want)
    del dbias, want
    # rows of 1 and -1 in turn: mean 0 and variance 1 without a rounding, so that unit is x / sqrt(1 + eps)
    rows, n = 2, (1 << 27) + 200
    x = torch.ones(rows, n, dtype=BF16, device=device)
    x[:, 1::2] = -1.0
    weight, bias = torch.ones(n, device=device, requires_grad=True), torch.zeros(n, device=device, requires_grad=True)
    dy = torch.ones(rows, n, dtype=BF16, device=device)
    odd = torch.tensor([1, 6, n // 2, (1 << 27) - 1, 1 << 27, n - 1], device=device)
    dy[1, odd] = 3.0
    dweight, dbias = torch.autograd.grad(tritonix.layer_norm(x, weight, bias), (weight, bias), dy)
    total = torch.full((n,), 2.0, device=device)
    total[odd] = 4.0
    assert torch.equal(dbias, total)
    # (the statistics: sums of n terms whose partial ones are whole numbers up to 2^18 a thread, then a tree of 1024 of them: 12 additions with a rounding each)
    unit = (1 + 1e-5) ** -0.5
    assert ((dweight.double() - total.double() * x[0].double() * unit).abs() <= 32 * ref.E * total).all()
