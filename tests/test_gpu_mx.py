"""Microscaled 4-bit tensors on the GPU: quantisation is the definition's bits, products stay within the error of 32-bit sums."""
import numpy as np
import pytest
import torch

import tritonix
from tests import mx_reference as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def make(shape, dtype, seed, scale=1.0):
    g = torch.Generator("cpu").manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def same(got, want):
    got = got.cpu().double().numpy()
    assert got.shape == want.shape
    np.testing.assert_array_equal(got, want)             # NaN equals NaN here


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim", [-1, -2])
@pytest.mark.parametrize("shape", [(1, 1), (1, 32), (3, 31), (5, 33), (2, 255), (129, 257), (64, 512), (130, 1000), (257, 129), (1, 5000),
                                   (5000, 1), (2, 33, 70), (3, 32, 256)], ids=str)
def test_round_trip_is_the_definition(device, dtype, dim, shape):
    x = make(shape, dtype, 1 + sum(shape), 3.0)
    t = tritonix.mx_quantize(x.to(device), dim=dim)
    assert t.shape == shape and t.t().shape == (*shape[:-2], shape[-1], shape[-2])
    same(tritonix.mx_dequantize(t, torch.float32), ref.values(x, dim))
    if dtype != torch.float16:                           # bfloat16 holds every such value
        same(tritonix.mx_dequantize(t, torch.bfloat16), ref.values(x, dim))


@pytest.mark.parametrize("dim", [-1, -2])
def test_every_rounding(device, dim):
    """Blocks of scale 1 (a 4 in each): every multiple of 1/64 up to 8 of either sign, so every tie and both its neighbours."""
    v = np.concatenate([s * np.arange(0, 512) / 64 for s in (1.0, -1.0)])
    v = np.concatenate([np.nextafter(v, -9, dtype=np.float32), v, np.nextafter(v, 9, dtype=np.float32)]).astype(np.float32)
    v = v[np.abs(v) < 8]
    v = np.concatenate([v, np.zeros(-len(v) % 31, np.float32)]).reshape(-1, 31)
    x = torch.from_numpy(np.concatenate([np.full((len(v), 1), 4.0, np.float32), v], axis=1))
    x = x if dim == -1 else x.t().contiguous()
    same(tritonix.mx_dequantize(tritonix.mx_quantize(x.to(device), dim=dim), torch.float32), ref.values(x, dim))


@pytest.mark.parametrize("dim", [-1, -2])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_extreme_blocks(device, dtype, dim):
    """Zeros of both signs, the smallest and largest numbers, infinities and NaN in one element of a block."""
    x = torch.zeros(12, 96)
    x[1] = -0.0
    x[2] = 2.0 ** -149 if dtype == torch.float32 else 2.0 ** -133
    x[3, 5], x[3, 6] = 1.5 * 2.0 ** -127, -2.0 ** -126
    x[4, ::3] = torch.finfo(dtype).max
    x[4, 1::3] = -2.0 ** 126
    x[5, 40] = float("inf")
    x[6, 70] = float("-inf")
    x[7, 31] = float("nan")
    x[7, 33] = 5.0
    x[8] = torch.exp2(torch.arange(96) - 60.0)
    x[9] = torch.finfo(dtype).tiny * 6
    x[10, 95] = 1e-30
    x = x.to(dtype)
    x = x if dim == -1 else x.t().contiguous()
    same(tritonix.mx_dequantize(tritonix.mx_quantize(x.to(device), dim=dim), torch.float32), ref.values(x, dim))


def test_codes_are_the_documented_bytes(device):
    """The two buffers byte by byte, and the padding: codes zero, scales 127 (rows past the last one excepted)."""
    rows, k = 37, 600
    x = make((rows, k), torch.bfloat16, 7)
    t = tritonix.mx_quantize(x.to(device))
    code, e, _ = ref.quantize(x.double().numpy())
    slabs = 3
    want = np.zeros((rows, slabs * 256), dtype=np.int64)
    want[:, :code.shape[1]] = code
    want = want[:, 0::2] + 16 * want[:, 1::2]
    np.testing.assert_array_equal(t.codes.cpu().numpy().reshape(rows, slabs * 128), want)
    scales = t.scales.cpu().numpy().reshape(2, 2, 32, 2, 8)       # row / 32, slab / 2, row % 32, slab % 2
    for r in range(rows):
        got = scales[r // 32, :, r % 32].reshape(-1)[:slabs * 8]
        np.testing.assert_array_equal(got[:19], e[r] + 127)
        assert (got[19:] == 127).all()


@pytest.mark.parametrize("k", [1, 31, 32, 63, 100, 256, 1000])
def test_from_codes(device, k):
    rows = 45
    g = torch.Generator("cpu").manual_seed(k)
    codes = torch.randint(0, 256, (rows, -(-k // 2)), generator=g, dtype=torch.uint8)
    scales = torch.randint(100, 150, (rows, -(-k // 32)), generator=g, dtype=torch.uint8)
    scales[3, 0] = 255
    nib = np.stack([codes.numpy() % 16, codes.numpy() // 16], axis=2).reshape(rows, -1)[:, :k]
    v = np.where(nib >= 8, -1.0, 1.0) * ref.LEVELS[nib % 8]
    s = np.exp2(scales.numpy().astype(np.float64) - 127)
    s[scales.numpy() == 255] = np.nan
    want = v * np.repeat(s, 32, axis=1)[:, :k]
    t = tritonix.MXTensor.from_codes(codes.to(device), scales.to(device), k)
    same(tritonix.mx_dequantize(t, torch.float32), want)
    batch = tritonix.MXTensor.from_codes(torch.stack([codes, codes.flip(0)]).to(device), torch.stack([scales, scales.flip(0)]).to(device), k, dim=-2)
    assert batch.shape == (2, k, rows)
    same(tritonix.mx_dequantize(batch, torch.float32), np.stack([want.T, want[::-1].T]))


@pytest.mark.parametrize("dim", [-1, -2])
def test_strided_and_unaligned_sources(device, dim):
    base = make((70, 300), torch.bfloat16, 3).to(device)
    for x in (base[1:, 1:], base[::2, ::3], base.t(), base[:, :257], base.t()[3:, 5:]):
        same(tritonix.mx_dequantize(tritonix.mx_quantize(x, dim=dim), torch.float32), ref.values(x, dim))


def check_product(out, a, b, dtype, k):
    want = a @ b
    tol = ref.product_bound(a, b, k)
    tol = tol + ref.rounding(np.abs(want) + tol, dtype)
    got = out.cpu().double().numpy()
    assert got.shape == want.shape and np.isfinite(got).all()
    worst = (np.abs(got - want) / tol).max()
    assert worst <= 1, worst


SIZES = [(1, 16, 32), (1, 1, 1), (3, 17, 31), (16, 64, 256), (17, 100, 300), (33, 130, 600), (64, 64, 64), (65, 257, 513), (100, 300, 1000),
         (200, 2000, 260), (257, 259, 2049), (1, 4096, 2048), (2, 300, 1000), (1, 130, 30720), (2, 70, 31000), (1, 20, 70000), (40, 50, 9000), (1000, 520, 777), (300, 4100, 512), (2049, 2100, 256), (3600, 3700, 300),
         (3, 20, 5000), (4, 70, 4096), (5, 300, 3000), (8, 257, 2048), (9, 33, 1700), (16, 100, 1024), (16, 40, 1025)]


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_product(device, size, dtype):
    m, n, k = size
    a, b = make((m, k), dtype, m + n, 2.0), make((k, n), dtype, k, 0.5)
    av, bv = ref.values(a, -1), ref.values(b, -2)
    out = tritonix.mx_matmul(a.to(device), tritonix.mx_quantize(b.to(device), dim=0))
    assert out.dtype == dtype and out.shape == (m, n)
    check_product(out, av, bv, dtype, k)


@pytest.mark.parametrize("size", [(1, 32, 64), (5, 70, 100), (40, 258, 300), (130, 514, 512), (400, 1026, 700), (2100, 2048, 260)], ids=str)
@pytest.mark.parametrize("activation", ["silu", "sigmoid", "none"])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_gated_product(device, size, activation, dtype):
    m, n, k = size
    a, b = make((m, k), torch.bfloat16, m), make((k, n), torch.bfloat16, n, 0.2)
    av, bv = ref.values(a, -1), ref.values(b, -2)
    z = av @ bv
    want, tol = ref.gated(z, ref.product_bound(av, bv, k), activation)
    tol = tol + ref.rounding(np.abs(want) + tol, dtype)
    out = tritonix.mx_glu(a.to(device), tritonix.mx_quantize(b.to(device), dim=0), activation, out_dtype=dtype)
    got = out.cpu().double().numpy()
    assert got.shape == (m, n // 2) and (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("m", [2, 40, 300])
def test_a_nan_block_reaches_its_row_or_column_only(device, m):
    n, k = 96, 320
    a, b = make((m, k), torch.bfloat16, 1), make((k, n), torch.bfloat16, 2)
    a[1, 300] = float("inf")
    b[100, 50] = float("nan")
    out = tritonix.mx_matmul(a.to(device), tritonix.mx_quantize(b.to(device), dim=0), out_dtype=torch.float32).cpu()
    bad = torch.isnan(out)
    want = torch.zeros(m, n, dtype=torch.bool)
    want[1] = True
    want[:, 50] = True
    assert torch.equal(bad, want)


def test_two_rows_of_a_wider_tensor(device):
    """Rows that the kernel quantises itself, with a stride and an odd start."""
    base, w = make((4, 700), torch.float32, 5), make((600, 200), torch.bfloat16, 6)
    q = tritonix.mx_quantize(w.to(device), dim=0)
    for dtype in TYPES:
        x = base.to(dtype)[1::2, 33:633]
        out = tritonix.mx_matmul(base.to(dtype).to(device)[1::2, 33:633], q, torch.float32)
        check_product(out, ref.values(x, -1), ref.values(w, -2), torch.float32, 600)


def test_empty_sizes(device):
    w = tritonix.mx_quantize(torch.ones(64, 32, device=device), dim=0)
    assert tritonix.mx_matmul(torch.ones(0, 64, device=device), w).shape == (0, 32)
    assert tritonix.mx_dequantize(tritonix.mx_quantize(torch.ones(0, 5, device=device))).shape == (0, 5)
    none = tritonix.mx_matmul(torch.ones(3, 0, device=device), torch.ones(0, 4, device=device))
    assert torch.equal(none.cpu(), torch.zeros(3, 4))


def test_repeated_calls_give_the_same_bits_on_any_stream(device):
    a, b = make((300, 1000), torch.bfloat16, 1).to(device), make((1000, 500), torch.bfloat16, 2).to(device)
    first = tritonix.mx_matmul(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        others = [tritonix.mx_matmul(a, b) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(first, o) for o in others)


def test_linear_gradients_are_the_formulas(device):
    m, k, n = 150, 200, 70
    x, w, dy = make((m, k), torch.bfloat16, 1), make((k, n), torch.bfloat16, 2, 0.3), make((m, n), torch.bfloat16, 3)
    xd, wd = x.to(device).requires_grad_(True), w.to(device).requires_grad_(True)
    y = tritonix.mx_linear(xd, wd)
    y.backward(dy.to(device))
    check_product(y.detach(), ref.values(x, -1), ref.values(w, -2), torch.bfloat16, k)
    check_product(xd.grad, ref.values(dy, -1), ref.values(w, -1).T, torch.bfloat16, n)
    check_product(wd.grad, ref.values(x, -2).T, ref.values(dy, -2), torch.bfloat16, m)


def test_linear_gradients_are_differences(device):
    """Operands that are 4-bit floats already, moved by a step to another such: the product is then linear in them and its
    differences are the gradient to the last bit."""
    m, k, n = 32, 64, 32
    g = torch.Generator("cpu").manual_seed(5)
    levels = torch.tensor([0.5, 1.0, 2.0, -1.0, -2.0, 3.0])
    pick = lambda *s: levels[torch.randint(0, 6, s, generator=g)]      # noqa: E731
    x, w, dy = pick(m, k), pick(k, n), pick(m, n)
    x[:, ::32] = 4.0
    x[::32, :] = 4.0                                     # every block of every direction has the scale 1
    w[::32, :] = 4.0
    w[:, ::32] = 4.0
    dy[:, ::32] = 4.0
    dy[::32, :] = 4.0
    xd, wd = x.to(device).requires_grad_(True), w.to(device).requires_grad_(True)
    y = tritonix.mx_linear(xd, wd)
    y.backward(dy.to(device))
    dyd = dy.to(device)
    for i, j in ((1, 1), (5, 40), (31, 63)):
        moved = x.clone()
        step = 1.0 if x[i, j] in (1.0, 2.0, 3.0) else -0.5 if x[i, j] in (-1.0,) else 0.5 if x[i, j] == 0.5 else -1.0
        moved[i, j] += step
        diff = (tritonix.mx_linear(moved.to(device), w.to(device)) - y.detach()) * dyd
        assert float(diff.double().sum()) / step == float(xd.grad[i, j])
    for i, j in ((1, 1), (40, 5), (63, 31)):
        moved = w.clone()
        step = 1.0 if w[i, j] in (1.0, 2.0, 3.0) else -0.5 if w[i, j] in (-1.0,) else 0.5 if w[i, j] == 0.5 else -1.0
        moved[i, j] += step
        diff = (tritonix.mx_linear(x.to(device), moved.to(device)) - y.detach()) * dyd
        assert float(diff.double().sum()) / step == float(wd.grad[i, j])


def test_a_weight_past_four_gigabytes(device):
    """5.1 GB of codes: the last rows' offsets do not fit 32 bits.  All codes 2 (value 1) with scale 1, the last row 4 (value 2), so the
    product with ones counts k."""
    from tritonix.ops.mx import MXTensor

    n, k = 80000, 131072
    w = MXTensor.empty(None, n, k, -2, device)
    w.codes.fill_(0x22)
    w.scales.fill_(127)
    w.codes[(n - 1) * (k // 2):].fill_(0x44)
    for m in (1, 40, 130):
        x = torch.ones(m, k, device=device, dtype=torch.bfloat16)
        out = tritonix.mx_matmul(x, w, out_dtype=torch.float32)
        assert bool((out[:, :-1] == k).all()) and bool((out[:, -1] == 2 * k).all())


def test_graph_replays_equal_the_eager_result(device):
    a, b = make((48, 512), torch.bfloat16, 1).to(device), tritonix.mx_quantize(make((512, 256), torch.bfloat16, 2).to(device), dim=0)
    eager = tritonix.mx_glu(a, b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = tritonix.mx_glu(a, b)
    for i in range(3):
        a2 = make((48, 512), torch.bfloat16, 10 + i).to(device)
        want = tritonix.mx_glu(a2, b)
        a.copy_(a2)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert eager.shape == out.shape
