"""dsv4cuda_grouped_gemm against 64-bit products. Tolerance: grouped_ref's bound of the fp32 sum,
and half a step of the output's type, 2^-8 or 2^-24 of the value."""
import pytest
import torch

import grouped_ref as ref

pytestmark = pytest.mark.gpu


def setup(counts, outs, width, fp8, seed=0, held=None):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rows = sum(counts)
    xq, xs = ref.activations(held or max(rows, 1), width, g)
    w, ws = (ref.fp8 if fp8 else ref.fp4)(len(counts), outs, width, g)
    offsets = torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32).cuda()
    return xq, xs, w, ws, offsets


def want(xq, xs, w, ws, offsets, src=None):
    """(products [rows][outs], their bound)."""
    x = ref.rows_of(xq, xs)
    edge = offsets.tolist()
    src = torch.arange(edge[-1], device="cuda") if src is None else src.long()
    there = (src >= 0) & (src < x.shape[0])
    x = torch.where(there[:, None], x[src.clamp(0, x.shape[0] - 1)], 0.0)
    y = torch.zeros(len(src), w.shape[1], dtype=torch.float64, device="cuda")
    b = torch.zeros_like(y)
    for e in range(w.shape[0]):
        a, z = edge[e], edge[e + 1]
        if a < z:
            v = ref.fp8_of(w[e], ws[e]) if w.shape[2] == xq.shape[1] else ref.fp4_of(w[e], ws[e])
            y[a:z] = x[a:z] @ v.T
            b[a:z] = ref.sum_bound(x[a:z], v)
    return y, b


def near(got, y, bound):
    half = 2.0 ** -8 if got.dtype is torch.bfloat16 else 2.0 ** -24
    d = (got.double() - y).abs()
    assert bool((d <= bound + half * (y.abs() + bound) + 1e-38).all()), float((d / (bound + 1e-30)).max())


CASES = [
    # counts, outs, width, fp8, bf16
    ([1], 128, 128, False, False),
    ([1], 1, 128, False, True),
    ([3, 0, 5], 256, 256, False, False),
    ([0, 0, 16, 17, 0], 129, 640, False, True),
    ([15, 96, 97, 1], 300, 384, False, False),
    ([192, 193, 400], 257, 512, False, True),
    ([1000, 3], 384, 1152, False, False),
    ([2] * 40, 64, 2048, False, False),
    ([700], 1000, 4096, False, True),
    ([1], 128, 128, True, False),
    ([33], 130, 896, True, True),
    ([5, 0, 250, 64], 256, 1024, True, False),
    ([2000], 520, 1024, True, True),
    ([1] * 6, 4096, 2048, False, True),
    ([64], 31, 7168, False, False),
]


@pytest.mark.parametrize("counts,outs,width,fp8,bf16", CASES)
def test_products(cuda, counts, outs, width, fp8, bf16):
    xq, xs, w, ws, offsets = setup(counts, outs, width, fp8)
    out = torch.full((sum(counts), outs), 7.0, dtype=torch.bfloat16 if bf16 else torch.float32,
                     device="cuda")
    cuda.grouped_gemm(out, xq, xs, w, ws, offsets)
    near(out, *want(xq, xs, w, ws, offsets))
    again = torch.empty_like(out)
    cuda.grouped_gemm(again, xq, xs, w, ws, offsets)
    assert torch.equal(out, again)  # whoever brings a tile's last part
    assert cuda.device_error() == 0


@pytest.mark.parametrize("fp8", [False, True])
def test_gather_and_scatter(cuda, fp8):
    counts = [20, 0, 130, 7]
    xq, xs, w, ws, offsets = setup(counts, 200, 384, fp8, held=50)
    n = sum(counts)
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    src = torch.randint(0, 50, (n,), dtype=torch.int32, device="cuda", generator=g)
    src[::9], src[4] = -1, 50           # no row of x: zeros
    dst = torch.randperm(n, device="cuda", generator=g).int() + 3
    dst[::11], dst[2] = -1, n + 10      # no row of out: left out
    wide = torch.full((n + 10, 333), 5.0, device="cuda")
    out = wide[:, :200]
    cuda.grouped_gemm(out, xq, xs, w, ws, offsets, src=src, dst=dst)
    y, b = want(xq, xs, w, ws, offsets, src)
    live = (dst >= 0) & (dst < n + 10)
    near(out[dst[live].long()], y[live], b[live])
    rest = torch.ones(n + 10, dtype=torch.bool, device="cuda")
    rest[dst[live].long()] = False
    assert bool((out[rest] == 5).all()) and bool((wide[:, 200:] == 5).all())


def test_offsets_that_are_none(cuda):
    """Descending or beyond n_rows: groups are empty, rows outside stay as they were."""
    xq, xs, w, ws, _ = setup([10, 10, 10], 130, 256, False)
    out = torch.full((30, 130), 5.0, device="cuda")
    offsets = torch.tensor([4, 9, 2, 200], dtype=torch.int32, device="cuda")
    cuda.grouped_gemm(out, xq, xs, w, ws, offsets)
    x = ref.rows_of(xq, xs)
    near(out[4:9], x[4:9] @ ref.fp4_of(w[0], ws[0]).T, ref.sum_bound(x[4:9], ref.fp4_of(w[0], ws[0])))
    near(out[9:], x[9:] @ ref.fp4_of(w[2], ws[2]).T, ref.sum_bound(x[9:], ref.fp4_of(w[2], ws[2])))
    assert bool((out[:4] == 5).all())
    offsets.zero_()
    out.fill_(5)
    cuda.grouped_gemm(out, xq, xs, w, ws, offsets)
    assert bool((out == 5).all())


@pytest.mark.parametrize("fp8", [False, True])
def test_scales_off_the_vector_boundary(cuda, fp8):
    xq, xs, w, ws, offsets = setup([40, 3], 200, 512, fp8)
    hold = torch.empty(ws.numel() + 64, dtype=torch.uint8, device="cuda")
    ws2 = hold[4:4 + ws.numel()].view(ws.shape).copy_(ws)
    hold2 = torch.empty(xs.numel() + 64, dtype=torch.uint8, device="cuda")
    xs2 = hold2[1:1 + xs.numel()].view(xs.shape).copy_(xs)
    out, two = torch.empty(43, 200, device="cuda"), torch.empty(43, 200, device="cuda")
    cuda.grouped_gemm(out, xq, xs, w, ws, offsets)
    cuda.grouped_gemm(two, xq, xs2, w, ws2, offsets)
    assert torch.equal(out, two)


def test_nan_codes_and_scales_stay_where_they_are(cuda):
    xq, xs, w, ws, offsets = setup([30, 20], 256, 384, False)
    xq[3, 200], xs[7, 1] = 0x7F, 255
    ws[1, 17, 5] = 255
    out = torch.empty(50, 256, device="cuda")
    cuda.grouped_gemm(out, xq, xs, w, ws, offsets)
    bad = torch.zeros(50, 256, dtype=torch.bool, device="cuda")
    bad[3], bad[7], bad[30:, 17] = True, True, True
    assert torch.equal(torch.isnan(out), bad)
    y, b = want(xq, xs, w, ws, offsets)
    near(out[~bad], y[~bad], b[~bad])


def test_extreme_scales(cuda):
    """Sums near both ends of fp32's range."""
    for code in (40, 200):
        xq, xs, w, ws, offsets = setup([20], 128, 256, False)
        ws.fill_(code)
        out = torch.empty(20, 128, device="cuda")
        cuda.grouped_gemm(out, xq, xs, w, ws, offsets)
        near(out, *want(xq, xs, w, ws, offsets))


def test_captured_and_on_streams(cuda):
    """A captured call follows offsets written after the capture; two streams with a workspace each
    do not meet."""
    counts = [50, 9, 70]
    xq, xs, w, ws, offsets = setup(counts, 300, 640, False)
    out = torch.zeros(129, 300, device="cuda")
    work = torch.empty(cuda.grouped_workspace_bytes(out, xq, w, 129), dtype=torch.uint8, device="cuda")
    cuda.grouped_gemm(out, xq, xs, w, ws, offsets, workspace=work)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cuda.grouped_gemm(out, xq, xs, w, ws, offsets, workspace=work)
    offsets.copy_(torch.tensor([0, 3, 100, 129], dtype=torch.int32))
    for _ in range(3):
        out.fill_(5)
        graph.replay()
        torch.cuda.synchronize()
        near(out, *want(xq, xs, w, ws, offsets))
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.empty_like(out) for _ in streams]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, o in zip(streams, outs):
            with torch.cuda.stream(s):
                cuda.grouped_gemm(o, xq, xs, w, ws, offsets)
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, out)


def test_capture_without_a_workspace_is_refused(cuda):
    xq, xs, w, ws, offsets = setup([5], 128, 128, False)
    out = torch.empty(5, 128, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(cuda.Dsv4CudaError, match="workspace"):
            cuda.grouped_gemm(out, xq, xs, w, ws, offsets)
        out.fill_(1)


@pytest.mark.parametrize("counts,outs,width,fp8,bf16", [
    ([i % 4 for i in range(1024)], 130, 256, False, True),    # more groups than threads
    ([0] * 700 + [5] + [0] * 200 + [40, 0], 257, 384, False, False),
    ([8], 1024, 4096, False, False),                          # few tiles: cut along the columns
    ([8], 1024, 2048, False, False),                          # or not
    ([300, 1, 1, 80, 17], 640, 3584, False, False),           # tiles of several sizes
    ([90, 16, 150], 2500, 1024, True, True),
])
def test_plans(cuda, counts, outs, width, fp8, bf16):
    xq, xs, w, ws, offsets = setup(counts, outs, width, fp8, seed=9)
    out = torch.full((sum(counts), outs), 7.0, dtype=torch.bfloat16 if bf16 else torch.float32, device="cuda")
    cuda.grouped_gemm(out, xq, xs, w, ws, offsets)
    near(out, *want(xq, xs, w, ws, offsets))
    again = torch.empty_like(out)
    cuda.grouped_gemm(again, xq, xs, w, ws, offsets)
    assert torch.equal(out, again) and cuda.device_error() == 0
