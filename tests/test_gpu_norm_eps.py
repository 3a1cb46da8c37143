"""norm_quant and PagedCache.write with an eps that is not small beside the mean of squares, over all
that the entries take: beyond fp32 together with the mean, and below what squares can hold. Against
64 bits, as in test_gpu_norm.py and test_gpu_paged_write.py."""
import pytest
import torch

import test_gpu_norm
import test_gpu_paged_write

pytestmark = pytest.mark.gpu


def scaled(n, width, dtype, scale):
    g = torch.Generator(device="cuda")
    g.manual_seed(n + width)
    x = torch.randn(n, width, device="cuda", generator=g).clamp(-4, 4)
    x = x / x.square().mean(dim=1, keepdim=True).sqrt()
    return (x * torch.tensor(scale, device="cuda")[:, None]).to(dtype)


# the mean of squares a little below and beyond fp32's limit (1.84e19 squared), and ordinary rows
LARGE = [1.7e19, 1.79e19, 2.5e19, 1.0, 1e18, 0.0, 3e25]
# squares that have few bits or none
SMALL = [1e-15, 3e-19, 1e-21, 4e-23, 1e-30, 0.0, 1.0]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("width", [96, 512, 7168])
@pytest.mark.parametrize("eps,scales", [(1e38, LARGE), (2.9e38, LARGE), (1e30, LARGE), (1e-29, SMALL),
                                        (1e-31, SMALL), (1e-38, SMALL), (1e-42, SMALL), (2e-45, SMALL)])
def test_norm(cuda, dtype, width, eps, scales):
    x = scaled(len(scales), width, dtype, scales)
    held = torch.tensor(eps, dtype=torch.float32).item()  # as the call takes it
    test_gpu_norm.check(cuda, x, None, None, eps=held)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("eps,scales", [(1e38, LARGE), (2.9e38, LARGE), (1e-29, SMALL), (1e-38, SMALL),
                                        (2e-45, SMALL)])
def test_write(cuda, dtype, eps, scales):
    pool = test_gpu_paged_write.pool_of(cuda, 16, 2)
    kv = scaled(len(scales), 512, dtype, scales)
    rows = torch.arange(len(scales), device="cuda") + 3
    gain = torch.ones(512, dtype=torch.bfloat16, device="cuda")
    before = test_gpu_paged_write.state(pool.caches[0])
    held = torch.tensor(eps, dtype=torch.float32).item()
    pool.write(0, kv, rows, gain=gain, eps=held)
    test_gpu_paged_write.check(before, test_gpu_paged_write.state(pool.caches[0]), kv, rows, gain, held,
                               None, None, 448, 32)
