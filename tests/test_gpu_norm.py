"""dsv4cuda_norm_quant against 64 bits. A thread adds at most 32 squares one after another and the
rest in a tree of 10: the mean errs by 42 2^-24, its root by half of that and the reciprocal root's
two units; with the sum x + residual and two products y errs by less than 28 2^-24 < 2^-19 of
itself. Codes may be any rounding of a value that near; out adds half a step of its type."""
import pytest
import torch

import grouped_ref as ref

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -19


def rows(n, width, dtype, g, scale=1.0, pad=0):
    return (torch.randn(n, width + pad, device="cuda", generator=g) * scale).to(dtype)[:, :width]


def check(cuda, x, gain, residual, with_sum=True, with_out=True, eps=1e-6):
    n, width = x.shape
    blocks = -(-width // 128)
    codes = torch.full((n + 1, width), 9, dtype=torch.uint8, device="cuda")
    scales = torch.full((n + 1, blocks), 9, dtype=torch.uint8, device="cuda")
    v = x.double() + (0 if residual is None else residual.double())
    sum_out = torch.empty(n, width, dtype=x.dtype, device="cuda") if with_sum else None
    out = torch.empty(n, width, dtype=x.dtype, device="cuda") if with_out else None
    cuda.norm_quant(x, gain, codes[:n], scales[:n], eps=eps, residual=residual, sum_out=sum_out, out=out)
    half = 2.0 ** -8 if x.dtype is torch.bfloat16 else 2.0 ** -24
    y = v / torch.sqrt((v * v).mean(dim=1, keepdim=True) + eps)
    y = y * (1 if gain is None else gain.double())
    if with_sum:
        assert bool(((sum_out.double() - v).abs() <= half * (1 + 2.0 ** -15) * v.abs()).all())
    if with_out:
        assert bool(((out.double() - y).abs() <= (half + EPS * (1 + half)) * y.abs() + 1e-38).all())
    low, high = ref.quantised_range(y, EPS * y.abs())
    s = ref.e8m0(scales[:n])
    for i, b in enumerate(y.split(128, dim=1)):
        top = b.abs().amax(dim=1)
        assert bool(((s[:, i] == ref.scale_of(top * (1 - EPS))) | (s[:, i] == ref.scale_of(top * (1 + EPS)))).all())
    got = ref.e4m3(codes[:n]) * s.repeat_interleave(128, dim=1)[:, :width]
    assert bool(((got >= low) & (got <= high)).all())
    assert bool((codes[n] == 9).all()) and bool((scales[n] == 9).all())
    return codes[:n], scales[:n]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,width,pad", [(1, 4096, 0), (5, 7168, 0), (3, 1, 0), (70, 16, 0), (9, 127, 3),
                                         (4, 129, 0), (130, 256, 8), (7, 1000, 5), (3, 2049, 7),
                                         (2, 16384, 0), (2, 32768, 0), (1, 20001, 0), (300, 8, 0)])
def test_rows(cuda, dtype, n, width, pad):
    g = torch.Generator(device="cuda")
    g.manual_seed(n + width)
    x = rows(n, width, dtype, g, pad=pad)
    gain = (1 + 0.2 * torch.randn(width, device="cuda", generator=g)).bfloat16()
    check(cuda, x, gain, rows(n, width, dtype, g, 3.0))
    check(cuda, x, None, None, with_sum=False, with_out=False)


def test_sum_in_place_and_strides(cuda):
    g = torch.Generator(device="cuda")
    g.manual_seed(0)
    for dtype in (torch.bfloat16, torch.float32):
        x, r = rows(33, 640, dtype, g, pad=24), rows(33, 640, dtype, g, pad=9)
        want = (x.float() + r.float()).to(dtype)
        codes = [torch.empty(33, 640, dtype=torch.uint8, device="cuda") for _ in range(3)]
        scales = [torch.empty(33, 5, dtype=torch.uint8, device="cuda") for _ in range(3)]
        cuda.norm_quant(x, None, codes[0], scales[0], residual=r)
        x2 = torch.empty(33, 700, dtype=dtype, device="cuda")[:, :640].copy_(x)
        cuda.norm_quant(x2, None, codes[1], scales[1], residual=r, sum_out=x2)
        assert torch.equal(x2, want)
        r2 = r.clone()
        cuda.norm_quant(x, None, codes[2], scales[2], residual=r2, sum_out=r2)
        assert torch.equal(r2, want)
        for c, s in zip(codes, scales):
            assert torch.equal(c, codes[0]) and torch.equal(s, scales[0])


def test_large_and_small_values(cuda):
    """Squares beyond fp32 in some rows and not in others; rows that eps alone norms; zeros."""
    g = torch.Generator(device="cuda")
    g.manual_seed(0)
    for width in (200, 4096):
        x = rows(12, width, torch.bfloat16, g).float()
        x *= torch.tensor([1e30, 1, 1e-20, 3e19, 1e-3, 2e38, 1, 1e18, 0, 1e25, 1e-30, 1], device="cuda")[:, None]
        x = x.clamp(-3e38, 3e38).bfloat16()
        check(cuda, x, None, None)


def test_rows_that_are_not_finite(cuda):
    g = torch.Generator(device="cuda")
    g.manual_seed(0)
    x = rows(6, 512, torch.float32, g)
    good = check(cuda, x, None, None)
    y = x.clone()
    y[1, 200], y[4, 5] = float("nan"), float("inf")
    codes = torch.empty(6, 512, dtype=torch.uint8, device="cuda")
    scales = torch.empty(6, 4, dtype=torch.uint8, device="cuda")
    cuda.norm_quant(y, None, codes, scales)
    for r in (0, 2, 3, 5):
        assert torch.equal(codes[r], good[0][r]) and torch.equal(scales[r], good[1][r])
    assert bool((scales[1] == 255).all())
    assert scales[4, 0].item() == 255 and bool((ref.e4m3(codes[4, 128:]) == 0).all())


def test_captured(cuda):
    g = torch.Generator(device="cuda")
    g.manual_seed(0)
    x = rows(8, 384, torch.bfloat16, g)
    codes, scales = torch.empty(8, 384, dtype=torch.uint8, device="cuda"), torch.empty(8, 3, dtype=torch.uint8, device="cuda")
    cuda.norm_quant(x, None, codes, scales)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cuda.norm_quant(x, None, codes, scales)
    x.copy_(rows(8, 384, torch.bfloat16, g))
    graph.replay()
    torch.cuda.synchronize()
    want = check(cuda, x, None, None)
    assert torch.equal(codes, want[0]) and torch.equal(scales, want[1])
