"""Route weights so large that they pass fp32 over a block's scale, where h itself is ordinary: gate and
up of activations that are small enough. Against 64 bits, as in test_gpu_moe_experts.py; a product of
gate and up below fp32's normal range adds 2^-149 of absolute error, times the weight 5e-7: far less
than the smallest step of blocks whose largest |h| is above 1 (2^-18)."""
import pytest
import torch

import grouped_ref as ref
from test_gpu_moe_experts import check, layer_of, routes

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 60, 700])
def test_huge_weights(cuda, n):
    layer, w = layer_of(cuda, 256, 256, 5, 2)
    g = torch.Generator(device="cuda")
    g.manual_seed(6)
    xq, xs = ref.activations(n, 256, g)
    idx, wt = routes(n, 5, 2)
    # gate and up are some 80 at scales of 1, 3e-19 at 2^-68, their product's half 4e-38
    xs[::2] = 127 - 68
    wt[::2] = torch.tensor([3e38, 1e38], device="cuda")
    check(cuda, layer, w, xq, xs, idx, wt)
    layer.close()
