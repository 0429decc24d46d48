"""norm_rotate of rows near both ends of the range whose squares fp32 holds."""
import pytest
import torch

from test_gpu_norm_rotate import compare, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [16, 256])
@pytest.mark.parametrize("size,eps", [(2e17, 1e-6), (2e17, 0.0), (1e-17, 0.0)])
def test_sizes_whose_squares_fit(dtype, d, size, eps):
    # (components of up to 5 times the size)
    x, dq, dk = inputs(1, 40, 2, 1, d, 2, d // 2, dtype)
    for n in "qk":
        x[n] = (x[n].float() * size).to(dtype)
    compare(x, dq, dk, eps=eps)
