"""dsv4cuda_beam_select against 64-bit log softmax. A row's sum of exponentials: 32 fp32 terms one
after another, each of an argument rounded to 24 bits (terms beyond e^-25 add nothing) and an
exponential good to 2^-22, 64 bits beyond: relative error below 107 2^-24 < 2^-17, which is the log's
absolute one. Candidates may be taken in another order only where their totals are that near; within
a beam, and between beams with equal rows, the order is exact."""
import pytest
import torch

pytestmark = pytest.mark.gpu
E = 2.0 ** -17


def select(cuda, logits, score, cands, eos=-1, slot=None, **kw):
    g, b = score.shape
    i32 = dict(dtype=torch.int32, device="cuda")
    parent, token = torch.full((g, cands), -9, **i32), torch.full((g, cands), -9, **i32)
    total = torch.full((g, cands), 9e9, device="cuda")
    nxt = torch.full((g, b), -9, **i32)
    dst = src = None
    if slot is not None:
        dst, src = torch.full((g, b), -9, **i32), torch.full((g, b), -9, **i32)
    cuda.beam_select(logits, score, parent, token, total, nxt, slot=slot, dst=dst, src=src, eos=eos, **kw)
    return parent, token, total, nxt, dst, src


def check(cuda, logits, score, cands, eos=-1, slot=None):
    g, b = score.shape
    vocab = logits.shape[1]
    parent, token, total, nxt, dst, src = (None if t is None else t.cpu() for t in
                                           select(cuda, logits, score, cands, eos, slot))
    x = logits.double().cpu().view(g, b, vocab)
    broken = torch.isnan(x).any(2) | (x == float("inf")).any(2) | ~torch.isfinite(score.double().cpu())
    lp = torch.log_softmax(x, dim=2)
    every = score.double().cpu()[:, :, None] + lp
    every[broken] = -float("inf")
    every = torch.where(torch.isnan(every), -float("inf"), every).view(g, -1)
    best = every.sort(dim=1, descending=True, stable=True)
    for i in range(g):
        n = min(cands, int((every[i] > -float("inf")).sum()))
        assert bool((parent[i, n:] == -1).all()) and bool((token[i, n:] == -1).all())
        assert bool((total[i, n:] == -float("inf")).all())
        place = parent[i, :n].long() * vocab + token[i, :n]
        assert len(set(place.tolist())) == n and bool((parent[i, :n] >= 0).all()) and bool((token[i, :n] >= 0).all())
        t = every[i][place]
        w = best.values[i, :n]
        assert bool(((t - w).abs() <= 2 * E).all())
        assert bool(((total[i, :n].double() - t).abs() <= E + 2.0 ** -24 * (t.abs() + E)).all())
        clear = torch.ones(n, dtype=torch.bool)  # positions that no near neighbour may take
        gap = (best.values[i, :-1] - best.values[i, 1:])[:n]
        near = (gap <= 2 * E) & (best.indices[i, :-1][:n] // vocab != best.indices[i, 1:][:n] // vocab)
        clear[:len(near)] &= ~near
        clear[1:] &= ~near[:n - 1]
        assert torch.equal(place[clear], best.indices[i, :n][clear])
        # who goes on
        on = [j for j in range(n) if token[i, j] != eos][:b]
        assert nxt[i].tolist() == on + [-1] * (b - len(on))
        if slot is not None:
            s = slot[i].tolist()
            mothers = [int(parent[i, j]) for j in on] + [-1] * (b - len(on))
            lost = [s[k] for k in range(b) if k not in mothers]
            for k, m in enumerate(mothers):
                stays = m >= 0 and m not in mothers[:k]
                assert dst[i, k].item() == (s[m] if stays else lost.pop(0))
                assert src[i, k].item() == (s[m] if m >= 0 else -1)
    return parent, token, total, nxt, dst, src


def rows(g, b, vocab, dtype, seed=0, pad=0, masked=0.0):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    x = torch.randn(g * b, vocab + pad, device="cuda", generator=gen) * 2.5
    if masked:
        x = torch.where(torch.rand(x.shape, device="cuda", generator=gen) < masked, -float("inf"), x)
    x[:, vocab:] = 1e30
    score = -torch.rand(g, b, device="cuda", generator=gen) * 5
    slot = torch.randperm(g * b, device="cuda", generator=gen).int().view(g, b)
    return x.to(dtype)[:, :vocab], score, slot


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("g,b,vocab,cands,pad,masked", [
    (1, 4, 129280, 8, 0, 0.0), (3, 8, 129280, 16, 8, 0.2), (2, 1, 1000, 1, 0, 0.0), (5, 32, 4099, 32, 1, 0.0),
    (2, 5, 100, 10, 3, 0.5), (4, 3, 7, 32, 0, 0.3), (1, 2, 1, 2, 0, 0.0), (3, 16, 8192, 31, 0, 0.95),
    (2, 6, 8193, 12, 0, 0.9995), (6, 2, 20000, 9, 5, 0.0)])
def test_select(cuda, dtype, g, b, vocab, cands, pad, masked):
    x, score, slot = rows(g, b, vocab, dtype, g + b, pad, masked)
    check(cuda, x, score, cands, slot=slot)
    eos = int(x[0].float().argmax())
    check(cuda, x, score, cands, eos=eos, slot=slot)


def test_beams_that_are_not_there(cuda):
    x, score, slot = rows(4, 4, 5000, torch.float32)
    score[0, 1:] = -float("inf")
    score[1] = -float("inf")
    score[2, 2] = float("nan")
    check(cuda, x, score, 8, slot=slot)


def test_rows_that_are_not_finite_or_masked_whole(cuda):
    x, score, slot = rows(4, 3, 9000, torch.float32)
    x[0, 77], x[4, 8999], x[7] = float("nan"), float("inf"), -float("inf")
    x[9:12] = -float("inf")
    x[10, 123] = 1.0
    parent, token, *_ = check(cuda, x, score, 6, slot=slot)
    assert parent[3, 0] == 1 and token[3, 0] == 123 and parent[3, 1] == -1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_equal_values_and_equal_beams(cuda, dtype):
    """Constant rows (more equal values than are held at once), equal beams: the lowest beam, then
    the lowest token, whatever the rows' alignment."""
    for vocab, pad in ((20000, 0), (20001, 0), (9001, 2)):
        x = torch.zeros(6, vocab + pad, dtype=dtype, device="cuda")[:, :vocab]
        score = torch.tensor([[-1.0, -1.0, -2.0], [-3.0, -0.5, -0.5]], device="cuda")
        parent, token, *_ = check(cuda, x, score, 8)
        assert token.tolist() == [list(range(8))] * 2
        assert parent.tolist() == [[0] * 8, [1] * 8]
        y, _, _ = rows(1, 1, vocab, dtype, 5)
        x.copy_(y.expand(6, vocab))
        score.fill_(-1.5)
        parent, token, *_ = check(cuda, x, score, 9)
        assert parent.tolist() == [[0, 1, 2] * 3] * 2
        assert bool((token.view(2, 3, 3) == token.view(2, 3, 3)[:, :, :1]).all())


def test_values_in_order(cuda):
    x = torch.arange(30000, device="cuda").float()[None].repeat(4, 1) * 1e-3
    x[1] = x[1].flip(0)
    score = torch.tensor([[-1.0, -2.0], [-2.0, -1.0]], device="cuda")
    check(cuda, x, score, 32)


def test_slots_with_fork(cuda):
    """dst and src through PagedCache.fork: every new beam's slot holds its parent's latents, and the
    pool keeps count."""
    b, page = 4, 4
    cache = cuda.LatentCache(40 * page)
    pool = cuda.PagedCache.empty([cache], page, 2 * b, 8)
    i32 = dict(dtype=torch.int32, device="cuda")
    slots, counts = torch.arange(2 * b, **i32), torch.tensor([5, 9, 8, 3, 6, 1, 4, 11], **i32)
    new = torch.empty(int(counts.sum()), dtype=torch.int64, device="cuda")
    pool.append(slots, counts, new)
    kv = torch.randn(len(new), 512, generator=torch.Generator().manual_seed(0)).bfloat16().cuda()
    pool.write(0, kv, new)

    def held(s):
        n = int(pool.length[s])
        at = torch.tensor([int(pool.table[s, p // page]) * page + p % page for p in range(n)], device="cuda")
        out = torch.empty(n, 512, device="cuda")
        cache.read(at, out)
        return out
    before = [held(s) for s in range(2 * b)]
    x, score, _ = rows(2, b, 500, torch.float32, 3)
    slot = torch.tensor([[4, 0, 7, 2], [1, 3, 6, 5]], **i32)
    parent, token, total, nxt, dst, src = select(cuda, x, score, 8, slot=slot)
    pool.fork(dst.flatten(), src.flatten())
    assert pool.status() == 0
    for i in range(2):
        assert sorted(dst[i].tolist()) == sorted(slot[i].tolist())
        for k in range(b):
            mother = int(parent[i, int(nxt[i, k])])
            assert torch.equal(held(int(dst[i, k])), before[int(slot[i, mother])])
    # every page's count is the entries that name it
    names = pool.table[pool.table >= 0].long()
    assert torch.equal(torch.bincount(names, minlength=40).int(), pool.refs)


def test_captured_and_on_streams(cuda):
    x, score, slot = rows(3, 5, 10000, torch.bfloat16)
    select(cuda, x, score, 10, slot=slot)
    i32 = dict(dtype=torch.int32, device="cuda")
    parent, token, total = torch.empty(3, 10, **i32), torch.empty(3, 10, **i32), torch.empty(3, 10, device="cuda")
    nxt, dst, src = (torch.empty(3, 5, **i32) for _ in range(3))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cuda.beam_select(x, score, parent, token, total, nxt, slot=slot, dst=dst, src=src)
    for seed in (7, 8):
        y, s, _ = rows(3, 5, 10000, torch.bfloat16, seed)
        x.copy_(y)
        score.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        want = check(cuda, x, score, 10, slot=slot)
        for a, w in zip((parent, token, total, nxt, dst, src), want):
            assert torch.equal(a.cpu(), w)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got += [select(cuda, x, score, 10, slot=slot) for _ in range(4)]
    torch.cuda.synchronize()
    for r in got:
        for a, w in zip(r, want):
            assert torch.equal(a.cpu(), w)


@pytest.mark.parametrize("beams", [5, 32])
def test_slots_in_place(cuda, beams):
    g = torch.Generator(device="cuda")
    g.manual_seed(11)
    x = torch.randn(4 * beams, 700, device="cuda", generator=g) * 3
    score = -torch.rand(4, beams, device="cuda", generator=g)
    slot = torch.randperm(4 * beams, device="cuda", generator=g).int().view(4, beams)
    i32 = dict(dtype=torch.int32, device="cuda")
    outs = []
    for dst in (torch.empty(4, beams, **i32), slot.clone()):
        at = slot if not outs else dst
        p, t, nxt, src = (torch.empty(4, n, **i32) for n in (beams, beams, beams, beams))
        total = torch.empty(4, beams, device="cuda")
        cuda.beam_select(x, score, p, t, total, nxt, slot=at, dst=dst, src=src)
        outs.append((p, t, total, nxt, dst, src))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
