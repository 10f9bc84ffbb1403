"""A matrix's dimensions are what they are called, of codes as of a tensor."""
import pytest
import torch

import tritonix

pytestmark = pytest.mark.gpu


def rand(device, *shape, dtype=torch.float32, seed=0):
    return torch.randn(shape, generator=torch.Generator("cpu").manual_seed(seed)).to(dtype).to(device)


@pytest.mark.parametrize("dim", [1, 2, -1, -2])
def test_a_batch_counts_its_dimensions_from_the_batch(device, dim):
    """from_codes as mx_quantize: of three dimensions 1 is the last but one and 2 the last."""
    x = rand(device, 2, 40, 70) if dim in (2, -1) else rand(device, 2, 70, 40)
    t = tritonix.mx_quantize(x, dim=dim)
    codes = torch.randint(0, 256, (2, 40, 35), generator=torch.Generator("cpu").manual_seed(1), dtype=torch.uint8).to(device)
    scales = torch.full((2, 40, 3), 127, dtype=torch.uint8, device=device)
    made = tritonix.MXTensor.from_codes(codes, scales, 70, dim=dim)
    assert made.shape == t.shape == tuple(x.shape) and made.dim == t.dim


def test_a_batch_has_no_codes_along_the_batch(device):
    codes, scales = torch.zeros(2, 4, 16, dtype=torch.uint8, device=device), torch.full((2, 4, 1), 127, dtype=torch.uint8, device=device)
    with pytest.raises(ValueError, match="dim 0"):
        tritonix.MXTensor.from_codes(codes, scales, 32, dim=0)
    for dim, shape in ((0, (32, 4)), (1, (4, 32)), (-1, (4, 32)), (-2, (32, 4))):
        assert tritonix.MXTensor.from_codes(codes[0], scales[0], 32, dim=dim).shape == shape
