"""PagedCache.write: latents normed, turned and quantised into their pages, against 64 bits. A lane
adds at most 18 squares one after another and five more roundings in a tree: with the root and the
products a value errs by less than 2^-19 of itself; a turned one by that of |a| + |b|. Codes may be
any rounding of a value that near, RoPE values add half a BF16 step, 2^-8."""
import pytest
import torch

import grouped_ref as ref

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -19


def pool_of(cuda, page, pages, nope=448, rope=64, layers=1, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    total = page * pages
    caches = []
    for _ in range(layers):
        codes = torch.randint(0, 127, (total, nope), dtype=torch.uint8, device="cuda", generator=g)
        scales = torch.randint(119, 123, (total, 8), dtype=torch.uint8, device="cuda", generator=g)
        rope_v = torch.randn(total, rope, device="cuda", generator=g).bfloat16().view(torch.int16)
        caches.append(cuda.LatentCache.from_tensors(codes, scales, rope_v))
    return cuda.PagedCache.empty(caches, page, 4, pages)


def state(cache):
    return cache.codes.clone(), cache.scales.clone(), cache.rope.clone()


def check(before, after, kv, rows, gain, eps, cos, sin, nope, limit):
    live = (rows >= 0) & (rows < limit)
    at = rows[live]
    v = kv.double()
    if gain is not None:
        v = v / torch.sqrt((v * v).mean(dim=1, keepdim=True) + eps) * gain.double()
    low, high = ref.quantised_range(v[:, :nope], EPS * v[:, :nope].abs(), 64)
    scale = ref.e8m0(after[1][at][:, :nope // 64])
    got = ref.e4m3(after[0][at]) * scale.repeat_interleave(64, dim=1)
    assert bool(((got >= low[live]) & (got <= high[live])).all())
    a, b = v[:, nope::2], v[:, nope + 1::2]
    y, size = torch.stack([a, b], 2).flatten(1), torch.stack([a.abs(), b.abs()], 2).flatten(1)
    if cos is not None:
        c, s = cos.double(), sin.double()
        y = torch.stack([a * c - b * s, a * s + b * c], 2).flatten(1)
        size = (a.abs() + b.abs()).repeat_interleave(2, dim=1)
    got = after[2].view(torch.bfloat16)[at].double()
    assert bool(((got - y[live]).abs() <= 2.0 ** -8 * y[live].abs() + 2 * EPS * size[live] + 1e-38).all())
    same = torch.ones(before[0].shape[0], dtype=torch.bool, device="cuda")
    same[at] = False
    for x, z in zip(before, after):
        assert torch.equal(x[same], z[same])
    assert torch.equal(before[1][:, nope // 64:], after[1][:, nope // 64:])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,page,nope,rope,normed,turned,pad", [
    (1, 16, 448, 64, True, True, 0), (37, 7, 448, 64, True, True, 0), (500, 64, 448, 64, False, True, 8),
    (130, 48, 448, 64, True, False, 3), (9, 16, 64, 16, True, True, 0), (21, 16, 512, 6, True, True, 1),
    (6, 5, 128, 200, False, True, 0), (5, 16, 64, 0, True, False, 0)])
def test_write(cuda, dtype, n, page, nope, rope, normed, turned, pad):
    pages = -(-n // page) + 3
    pool = pool_of(cuda, page, pages, nope, rope, layers=2)
    g = torch.Generator(device="cuda")
    g.manual_seed(n)
    d = nope + rope
    kv = (torch.randn(n, d + pad, device="cuda", generator=g) * 2).to(dtype)[:, :d]
    rows = torch.randperm(page * pages, device="cuda", generator=g)[:n]
    if n > 5:
        rows[3], rows[n - 1] = -1, page * pages  # no row of a page
    gain = (1 + 0.2 * torch.randn(d, device="cuda", generator=g)).bfloat16() if normed else None
    angle = torch.rand(n, rope // 2, device="cuda", generator=g) * 6
    cos, sin = (angle.cos(), angle.sin()) if turned else (None, None)
    before = [state(c) for c in pool.caches]
    pool.write(1, kv, rows, gain=gain, eps=1e-5, rope_cos=cos, rope_sin=sin)
    for x, z in zip(before[0], state(pool.caches[0])):
        assert torch.equal(x, z)
    check(before[1], state(pool.caches[1]), kv, rows, gain, 1e-5, cos, sin, nope, page * pages)


def test_as_the_caches_own_write(cuda):
    """Without norm and rotation, BF16 values become what LatentCache.write makes of them."""
    pool = pool_of(cuda, 16, 20, layers=2)
    kv = (torch.randn(300, 512, generator=torch.Generator().manual_seed(1)) * 5).bfloat16().cuda()
    kv[5], kv[6, :64], kv[7] = 0, -0.0, 3e38
    kv[8, 70] = 1e-30
    rows = torch.randperm(320, device="cuda")[:300]
    rows[17] = -1
    pool.caches[1].codes.copy_(pool.caches[0].codes)
    pool.caches[1].scales.copy_(pool.caches[0].scales)
    pool.caches[1].rope.copy_(pool.caches[0].rope)
    pool.caches[0].write(kv.float(), rows)
    pool.write(1, kv, rows)
    for x, z in zip(state(pool.caches[0]), state(pool.caches[1])):
        assert torch.equal(x, z)


def test_latents_that_are_not_finite(cuda):
    """A group with a NaN or infinity is NaN to its reader; the attention of rows that do not see it
    is what it was."""
    pool = pool_of(cuda, 16, 4)
    kv = torch.randn(40, 512, generator=torch.Generator().manual_seed(1)).cuda()
    kv[20, 3], kv[30, 500] = float("inf"), float("nan")
    rows = torch.empty(40, dtype=torch.int64, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    pool.append(torch.zeros(1, **i32), torch.full((1,), 40, **i32), rows)
    pool.write(0, kv, rows)
    q = torch.randn(40, 8, 512, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    out = torch.empty_like(q)
    cuda.paged_attn(out, q, pool, 0, torch.tensor([0, 40, 40, 40, 40], **i32), 40, 40, 0.05)
    bad = torch.isnan(out).flatten(1).any(dim=1)
    assert bad.tolist() == [False] * 20 + [True] * 20


def test_normed_rows_with_large_values(cuda):
    pool = pool_of(cuda, 16, 2)
    kv = torch.randn(3, 512, generator=torch.Generator().manual_seed(1)).cuda()
    kv *= torch.tensor([1e25, 1.0, 3e37], device="cuda")[:, None]
    rows = torch.arange(3, device="cuda")
    gain = torch.ones(512, dtype=torch.bfloat16, device="cuda")
    before = state(pool.caches[0])
    pool.write(0, kv, rows, gain=gain)
    check(before, state(pool.caches[0]), kv, rows, gain, 1e-6, None, None, 448, 32)


def test_captured_after_an_append(cuda):
    """A captured step: append gives the rows, write fills them, on tables that change between
    replays."""
    pool = pool_of(cuda, 8, 20)
    i32 = dict(dtype=torch.int32, device="cuda")
    slots, counts = torch.tensor([0, 2], **i32), torch.tensor([3, 5], **i32)
    rows = torch.empty(12, dtype=torch.int64, device="cuda")
    kv = torch.randn(12, 512, generator=torch.Generator().manual_seed(1)).cuda()
    gain = torch.ones(512, dtype=torch.bfloat16, device="cuda")
    def step():
        pool.append(slots, counts, rows)
        pool.write(0, kv, rows, gain=gain)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for n in ((3, 5), (6, 6), (1, 0)):
        counts.copy_(torch.tensor(n, dtype=torch.int32))
        before = state(pool.caches[0])
        kv.copy_(torch.randn(12, 512, generator=torch.Generator().manual_seed(sum(n))))
        graph.replay()
        torch.cuda.synchronize()
        assert int((rows >= 0).sum()) == sum(n)
        check(before, state(pool.caches[0]), kv, rows, gain, 1e-6, None, None, 448, 160)
    assert pool.status() == 0
