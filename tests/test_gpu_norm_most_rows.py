"""norm_quant of as many rows as an int counts."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_most_rows(cuda):
    """Rows of one value: y = 1 to fp32's rounding whatever the value is, 256 times the scale 2^-8."""
    n = (1 << 31) - 1
    x = torch.full((n, 1), 2.0, dtype=torch.bfloat16, device="cuda")
    x[-1], x[-2], x[0] = 1e4, -3.0, 0.5
    codes = torch.zeros(n, 1, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(n, 1, dtype=torch.uint8, device="cuda")
    cuda.norm_quant(x, None, codes, scales, eps=1e-12)
    del x
    assert bool((scales == 119).all())
    codes[-2] ^= 0x80
    assert bool((codes == 0x78).all())
