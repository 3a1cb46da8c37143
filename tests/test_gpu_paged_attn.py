"""dsv4cuda_paged_attn against attention in 64 bits, row by row.

Tolerances. Let A_i = sum_t p_t |v_t,i| with p the exact weights (after the
inverse RoPE, whose pairs mix, A of a pair is |cos| A_0 + |sin| A_1).
- A weight held in BF16 is off by at most 2^-9 of itself, the output's
  rounding by 2^-9 of the output: together at most 2^-8 A.
- Scores are fp32 sums of 512 products (exact each): with X = scale *
  max_t sum_i |q_i k_t,i| a score is off by at most dx = 2^-24 * 512 * X
  (the tensor core adds in another order, and may drop the bits of an addend
  below the largest one's last place, one more 2^-24 X per addition: 2 dx).
  A weight then moves by 2 dx of itself, and so does the denominator: 4 dx
  A in all. lse moves by 2 dx.
- exp2 is good to 2^-22, a sum of n weights in fp32 to 2^-24 n / 8 (partial
  sums): below 2^-11 for every length here.
So |got - want| <= (2^-8 + 4 dx + 2^-11) A and |lse - want| <= 2 dx +
2^-11 / 16 + 2^-22 |want|; the general kernel keeps its weights in fp32 and
is inside the same bound."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def latents(rng, rows, nope, rope):
    """Random cache contents and their values [rows][nope + rope] in float64."""
    codes = torch.from_numpy(rng.normal(size=(rows, nope)).astype(np.float32) * 100)
    codes = codes.clamp(-448, 448).to(torch.float8_e4m3fn)
    scales = torch.from_numpy(rng.integers(117, 123, (rows, 8)).astype(np.uint8))
    r = torch.from_numpy(rng.normal(size=(rows, rope)).astype(np.float32)).bfloat16()
    value = codes.double().view(rows, nope // 64, 64) * (
        2.0 ** (scales[:, :nope // 64].double() - 127))[:, :, None]
    return codes.view(torch.uint8), scales, r, torch.cat([value.flatten(1), r.double()], 1)


class Case:
    """Sequences of (new, length) over randomly placed pages."""

    def __init__(self, cuda, seqs, heads, page=64, window=0, nope=448, rope=64, bf16=True,
                 freed=False, seed=0, layers=1, spread=1.5, pad=0):
        rng = np.random.default_rng(seed)
        self.cuda, self.seqs, self.heads, self.page, self.window = cuda, seqs, heads, page, window
        self.dim, self.rope = nope + rope, rope
        held = [-(-length // page) for _, length in seqs]
        width = max(held) + 2
        pages = sum(held) + 2
        order = rng.permutation(pages).tolist()
        self.table = np.full((len(seqs), width), -1)
        for s, h in enumerate(held):
            first = 0
            if freed and window:
                n, length = seqs[s]
                first = max(0, length - n - window + 1) // page
            for j in range(first, h):
                self.table[s, j] = order.pop()
        caches = []
        for _ in range(layers):
            codes, scales, r, self.value = latents(rng, pages * page, nope, rope)
            caches.append(cuda.LatentCache.from_tensors(codes.cuda(), scales.cuda(),
                                                        r.cuda().view(torch.int16)))
        self.layer = layers - 1
        i32 = dict(dtype=torch.int32, device="cuda")
        refs = np.bincount(self.table[self.table >= 0], minlength=pages)
        self.pool = cuda.PagedCache(caches, page, torch.tensor(self.table, **i32),
                                    torch.tensor([b for _, b in seqs], **i32),
                                    torch.tensor(refs, **i32))
        self.starts = np.concatenate([[0], np.cumsum([n for n, _ in seqs])])
        self.q_start = torch.tensor(self.starts, **i32)
        total = int(self.starts[-1])
        dtype = torch.bfloat16 if bf16 else torch.float32
        wide = heads * self.dim + pad
        self.q = torch.from_numpy((rng.normal(size=(total, wide)) * spread).astype(np.float32))
        self.q = self.q.bfloat16().to(dtype).cuda()[:, :heads * self.dim].view(
            total, heads, self.dim)
        self.out = torch.full((total, wide), 77.0, dtype=dtype, device="cuda")[
            :, :heads * self.dim].view(total, heads, self.dim)
        self.lse = torch.full((total, heads), 77.0, device="cuda")
        self.sink = torch.from_numpy(rng.normal(size=heads).astype(np.float32)).cuda()
        angle = torch.from_numpy(rng.uniform(0, 6.28, (total, rope // 2)).astype(np.float32))
        self.cos, self.sin = angle.cos().cuda(), angle.sin().cuda()
        self.scale = self.dim ** -0.5
        self.use_sink = self.use_rope = True

    def run(self, **kw):
        args = dict(sink=self.sink if self.use_sink else None, window=self.window,
                    rope_cos=self.cos if self.use_rope else None,
                    rope_sin=self.sin if self.use_rope else None, lse=self.lse)
        args.update(kw)
        self.cuda.paged_attn(self.out, self.q, self.pool, self.layer, self.q_start,
                             max(n for n, _ in self.seqs), max(b for _, b in self.seqs),
                             self.scale, **args)

    def visible(self, s, i):
        n, length = self.seqs[s]
        p = length - n + i
        t = np.arange(max(0, p - self.window + 1) if self.window else 0, p + 1)
        q = self.table[s, t // self.page]
        return (q * self.page + t % self.page)[q >= 0]

    def check(self, rows=None):
        torch.cuda.synchronize()
        got, lse = self.out.double().cpu().numpy(), self.lse.double().cpu().numpy()
        value, q = self.value.numpy(), self.q.double().cpu().numpy()
        sink = self.sink.double().cpu().numpy()
        cos, sin = self.cos.double().cpu().numpy(), self.sin.double().cpu().numpy()
        worst = 0.0
        for s, (n, _) in enumerate(self.seqs):
            for i in range(n):
                r = self.starts[s] + i
                if rows is not None and r not in rows:
                    continue
                k = value[self.visible(s, i)]
                bad = not np.isfinite(k).all()
                if bad:
                    assert np.isnan(got[r]).all() and np.isnan(lse[r]).all(), r
                    continue
                x = q[r] @ k.T * self.scale
                X = float((np.abs(q[r]) @ np.abs(k).T).max(initial=0) * self.scale)
                full = np.concatenate([x, sink[:, None]], 1) if self.use_sink else x
                if full.shape[1] == 0:
                    assert (got[r] == 0).all() and np.isneginf(lse[r]).all()
                    continue
                m = full.max(1, keepdims=True)
                e = np.exp(full - m)
                den = e.sum(1, keepdims=True)
                p = (e / den)[:, :k.shape[0]]
                want, A = p @ k, p @ np.abs(k)
                if self.use_rope:
                    c, sn = cos[r][None], sin[r][None]
                    a, b = want[:, -self.rope::2].copy(), want[:, 1 - self.rope::2].copy() \
                        if self.rope > 1 else None
                    Aa, Ab = A[:, -self.rope::2].copy(), A[:, 1 - self.rope::2].copy()
                    want[:, -self.rope::2], want[:, 1 - self.rope::2] = a * c + b * sn, b * c - a * sn
                    A[:, -self.rope::2] = np.abs(c) * Aa + np.abs(sn) * Ab
                    A[:, 1 - self.rope::2] = np.abs(c) * Ab + np.abs(sn) * Aa
                dx = 2.0 ** -24 * 512 * X
                tol = (2.0 ** -8 + 4 * dx + 2.0 ** -11) * A + 1e-30
                ratio = (np.abs(got[r] - want) / tol).max()
                assert ratio <= 1, (r, ratio)
                worst = max(worst, ratio)
                want_lse = (m + np.log(den))[:, 0]
                assert (np.abs(lse[r] - want_lse)
                        <= 2 * dx + 2.0 ** -15 + 2.0 ** -22 * np.abs(want_lse)).all(), r
        assert self.pool.status() == 0
        return worst


SEQS = {
    "one token": [(1, 1)],
    "tokens": [(1, 1), (1, 63), (1, 64), (1, 65), (1, 700)],
    "chunk from nothing": [(130, 130)],
    "chunk on top": [(67, 515)],
    "ragged": [(1, 300), (129, 129), (0, 50), (6, 1000), (33, 40), (0, 0)],
    "long": [(3, 9001)],
}


@pytest.mark.parametrize("heads", [64, 128])
@pytest.mark.parametrize("seqs", list(SEQS))
def test_lengths(cuda, seqs, heads):
    c = Case(cuda, SEQS[seqs], heads, seed=heads + len(seqs))
    c.run()
    c.check()


@pytest.mark.parametrize("heads", [1, 3, 16, 48, 100, 127])
def test_head_counts(cuda, heads):
    c = Case(cuda, [(5, 90), (1, 200), (40, 41)], heads, page=16, seed=heads)
    c.run()
    c.check()


@pytest.mark.parametrize("page", [1, 7, 48, 100, 512])
def test_page_sizes(cuda, page):
    c = Case(cuda, [(20, 333), (1, 130), (9, 9)], 64, page=page, seed=page)
    c.run()
    c.check()


@pytest.mark.parametrize("window", [1, 2, 63, 64, 128, 1000])
@pytest.mark.parametrize("freed", [False, True])
def test_windows(cuda, window, freed):
    c = Case(cuda, [(70, 400), (1, 777), (200, 200), (6, 129)], 64, page=16, window=window,
             freed=freed, seed=window)
    c.run()
    c.check()


@pytest.mark.parametrize("use_sink", [False, True])
@pytest.mark.parametrize("use_rope", [False, True])
def test_optional_inputs(cuda, use_sink, use_rope):
    c = Case(cuda, [(9, 100), (1, 64)], 64, seed=3)
    c.use_sink, c.use_rope = use_sink, use_rope
    c.run()
    c.check()
    c.run(lse=None)


@pytest.mark.parametrize("use_sink", [False, True])
def test_rows_that_see_nothing(cuda, use_sink):
    """Every page given back, or only the ones that some of the tokens see."""
    c = Case(cuda, [(3, 50), (40, 100), (1, 64)], 64, page=16, window=20, seed=5)
    c.use_sink = use_sink
    c.table[0] = -1
    c.table[1, 3:5] = -1        # positions 48 .. 79: tokens 67 .. 79 see nothing
    c.table[2, 3] = 10 ** 9     # not a page: nothing
    c.pool.table.copy_(torch.from_numpy(c.table).int())
    c.table[2, 3] = -1
    c.run()
    c.check()


@pytest.mark.parametrize("bf16", [False, True])
def test_strides_and_types(cuda, bf16):
    c = Case(cuda, [(17, 90), (1, 300)], 64, bf16=bf16, pad=24, seed=7, layers=3)
    around = c.out.untyped_storage().nbytes()
    c.run()
    c.check()
    assert c.out.untyped_storage().nbytes() == around
    whole = torch.as_strided(c.out, (18, 64 * 512 + 24), (64 * 512 + 24, 1))
    assert (whole[:, 64 * 512:] == 77).all()            # what lies between the rows stays


@pytest.mark.parametrize("nope,rope,heads", [(64, 16, 4), (128, 64, 130), (448, 64, 200),
                                             (64, 6, 3), (512, 64, 8), (448, 32, 64)])
def test_other_shapes(cuda, nope, rope, heads):
    c = Case(cuda, [(5, 70), (1, 33), (20, 20)], heads, page=9, nope=nope, rope=rope, seed=nope)
    c.run()
    c.check()


@pytest.mark.parametrize("nope,rope", [(448, 64), (64, 16)])
@pytest.mark.parametrize("what", ["code", "scale", "rope nan", "rope inf", "overflow"])
def test_broken_latents_reach_only_who_sees_them(cuda, nope, rope, what):
    """NaN and infinities at positions behind a window, ahead of a token, in
    unused rows of the last page and in pages of nobody; and one that is seen."""
    c = Case(cuda, [(60, 200), (1, 130)], 16, page=16, window=50, nope=nope, rope=rope, seed=11)
    cache = c.pool.caches[0]

    def spoil(s, t):
        r = c.table[s, t // 16] * 16 + t % 16 if s is not None else t
        if what == "code":
            cache.codes[r, 5] = 0x7F
        elif what == "scale":
            cache.scales[r, 0] = 255
        elif what == "overflow":
            cache.scales[r, 0], cache.codes[r, 3] = 254, 0x7E
        else:
            cache.rope[r, 1] = 0x7FC0 if what == "rope nan" else 0x7F80
        c.value[r, 0] = math.nan
    spoil(0, 30)                # behind every token's window
    spoil(0, 180)               # seen by tokens 180 .. 199 only
    spoil(0, 91 + 0)            # in the window of position 140 alone
    spoil(1, 131 + 3)           # in the last page, behind the last position
    free = [q for q in range(c.pool.n_pages) if q not in c.table]
    spoil(None, free[0] * 16)
    c.run()
    c.check()
    assert torch.isnan(c.out[40:60]).all() and torch.isnan(c.out[0]).all()
    assert not torch.isnan(c.out[1:40]).any() and not torch.isnan(c.out[60:]).any()


def test_extreme_scales_of_the_cache(cuda):
    """Scale codes at the ends of their range: tiny and huge latents."""
    c = Case(cuda, [(4, 70)], 64, seed=13, spread=1.0)
    cache = c.pool.caches[0]
    cache.scales[:, 0] = 1
    cache.scales[:, 1] = 0
    cache.scales[:, 2] = 8
    cache.scales[:, 3] = 135
    v = cache.codes.view(torch.float8_e4m3fn).cpu().double().view(-1, 7, 64)
    # as the cache holds them: rounded to BF16 where that has fewer bits
    value = v * (2.0 ** (cache.scales[:, :7].cpu().double() - 127))[:, :, None]
    c.value[:, :448] = value.flatten(1).float().bfloat16().double()
    c.q[:, :, 192:256] *= 2.0 ** -8
    c.run()
    c.check()


def test_masks_of_a_chunk_do_not_leak(cuda):
    """A token's output is the same whatever later positions hold."""
    a = Case(cuda, [(150, 300)], 64, seed=17)
    a.run()
    first = a.out.clone()
    cache = a.pool.caches[0]
    t = np.arange(200, 300)
    r = torch.from_numpy(a.table[0, t // 64] * 64 + t % 64).cuda()
    cache.codes[r] = torch.randint(0, 120, cache.codes[r].shape, device="cuda", dtype=torch.uint8)
    a.run()
    assert torch.equal(a.out[:50], first[:50])
    assert not torch.equal(a.out[60:], first[60:])


def test_same_bits_every_time_and_split_does_not_show(cuda):
    c = Case(cuda, [(1, 5000), (3, 900)], 64, seed=19)
    c.run()
    a, b = c.out.clone(), c.lse.clone()
    for _ in range(3):
        c.run()
        assert torch.equal(a, c.out) and torch.equal(b, c.lse)
    c.run(max_keys=5900)
    c.check()


def test_merging_two_parts_by_lse(cuda):
    """Attention over all positions equals the lse-weighted sum over a window
    and what lies before it (the table's other pages)."""
    c = Case(cuda, [(1, 512)], 64, page=64, seed=23)
    c.use_sink = c.use_rope = False
    c.run()
    whole, lse = c.out.double().clone(), c.lse.double().clone()
    keep = c.pool.table.clone()
    parts = []
    for cut in (slice(0, 5), slice(5, None)):
        c.pool.table.copy_(keep)
        c.pool.table[0, cut] = -1
        c.run()
        parts.append((c.out.double().clone(), c.lse.double().clone()))
    m = torch.logaddexp(parts[0][1], parts[1][1])
    assert (m - lse).abs().max().item() < 1e-4
    both = sum(o * torch.exp(x - m)[..., None] for o, x in parts)
    assert (both - whole).norm() / whole.norm() < 2.0 ** -7


def test_streams_and_capture(cuda):
    c = Case(cuda, [(2, 130), (1, 700)], 64, seed=29)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.run()
    torch.cuda.current_stream().wait_stream(side)
    c.check()
    want = c.out.clone()
    c.out.zero_()
    need = cuda.paged_attn_workspace_bytes(c.q, c.pool, 2, 700)
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.run(workspace=ws)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(c.out, want)
    # the lengths live on the device: the graph follows them
    c.pool.length[1] = 600
    c.seqs[1] = (1, 600)
    g.replay()
    c.check()


def test_long_sequence_far_apart_in_a_large_pool(cuda):
    """Cache offsets past 2^31 bytes."""
    page, pages = 64, 80_000                     # 5.1 M rows: 2.3 GB of codes
    cache = cuda.LatentCache(page * pages)
    rng = np.random.default_rng(31)
    seqs = [(2, 1000)]
    c = Case(cuda, seqs, 64, page=page, seed=31)
    where = rng.choice(np.arange(pages - 20000, pages), c.table.shape[1], replace=False)
    small = c.pool.caches[0]
    for j in range(16):
        a, b = int(c.table[0, j]) * page, int(where[j]) * page
        for x, y in ((cache.codes, small.codes), (cache.scales, small.scales),
                     (cache.rope, small.rope)):
            x[b:b + page] = y[a:a + page]
    table = torch.full_like(c.pool.table, -1)
    table[0, :16] = torch.from_numpy(where[:16]).int()
    c.pool = cuda.PagedCache([cache], page, table, c.pool.length,
                             torch.zeros(pages, dtype=torch.int32, device="cuda"))
    c.run()
    c.check()


def test_refusals(cuda):
    c = Case(cuda, [(2, 30)], 64, seed=37)
    with pytest.raises(ValueError):
        cuda.paged_attn(c.out.float(), c.q, c.pool, 0, c.q_start, 2, 30, 1.0)
    with pytest.raises(ValueError):
        cuda.paged_attn(c.out.half(), c.q.half(), c.pool, 0, c.q_start, 2, 30, 1.0)
    with pytest.raises(ValueError):
        cuda.paged_attn(c.out, c.q.transpose(0, 1), c.pool, 0, c.q_start, 2, 30, 1.0)
    with pytest.raises(ValueError):
        cuda.paged_attn(c.out, c.q, c.pool, 0, c.q_start.long(), 2, 30, 1.0)
    with pytest.raises(ValueError):
        cuda.paged_attn(c.out, c.q, c.pool, 0, c.q_start[:1], 2, 30, 1.0)
    with pytest.raises(ValueError):
        cuda.paged_attn(c.out, c.q, c.pool, 0, c.q_start, 2, 30, 1.0, sink=c.sink[:5])
    with pytest.raises(cuda.Dsv4CudaError):
        cuda.paged_attn(c.out, c.q, c.pool, 1, c.q_start, 2, 30, 1.0)
    with pytest.raises(cuda.Dsv4CudaError):
        cuda.paged_attn(c.out, c.q, c.pool, 0, c.q_start, 2, 30, 1.0, rope_cos=c.cos)
    with pytest.raises(cuda.Dsv4CudaError):
        cuda.paged_attn(c.out, c.q, c.pool, 0, c.q_start, 2, 30, 1.0, window=-1)
    with pytest.raises(cuda.Dsv4CudaError, match="head_dim"):
        cuda.paged_attn(c.out[..., :256].contiguous(), c.q[..., :256].contiguous(), c.pool, 0,
                        c.q_start, 2, 30, 1.0)
    odd = torch.zeros(2 * 64 * 512 + 4, dtype=torch.bfloat16, device="cuda")[4:].view(2, 64, 512)
    with pytest.raises(cuda.Dsv4CudaError, match="aligned"):
        cuda.paged_attn(odd, c.q, c.pool, 0, c.q_start, 2, 30, 1.0)
    c.run()                                       # still usable
    c.check()


@pytest.mark.parametrize("nope,rope", [(448, 64), (64, 16)])
@pytest.mark.parametrize("max_new,max_len", [(4, 400), (5, 199), (5, 399), (4, 199)])
def test_slots_beyond_the_bounds(cuda, nope, rope, max_new, max_len):
    """A slot with more tokens, or a longer one, than was said: NaN and a
    status bit; the others are not touched by it."""
    c = Case(cuda, [(3, 100), (5, 200), (1, 400), (2, 64)], 16, page=16, nope=nope, rope=rope,
             seed=41)
    cuda.paged_attn(c.out, c.q, c.pool, 0, c.q_start, max_new, max_len, c.scale, sink=c.sink,
                    rope_cos=c.cos, rope_sin=c.sin, lse=c.lse)
    assert c.pool.status() == 4
    c.pool.status_word.zero_()
    bad = [r for s, (n, length) in enumerate(c.seqs) if n > max_new or length > max_len
           for r in range(c.starts[s], c.starts[s + 1])]
    assert torch.isnan(c.out[bad]).all() and torch.isnan(c.lse[bad]).all()
    c.check(rows=set(range(11)) - set(bad))


def test_more_keys_than_the_workspace_was_made_for(cuda):
    c = Case(cuda, [(2, 100), (1, 3000), (0, 0)], 64, seed=43)
    for last, fits in ((3000, False), (1500, True)):
        c.pool.length[1] = last
        c.seqs[1] = (1, last)
        c.out.fill_(77.0)
        cuda.paged_attn(c.out, c.q, c.pool, 0, c.q_start, 2, 3000, c.scale, sink=c.sink,
                        rope_cos=c.cos, rope_sin=c.sin, lse=c.lse, max_keys=1600)
        assert c.pool.status() == (0 if fits else 4)
        c.pool.status_word.zero_()
        if not fits:
            assert torch.isnan(c.out[2]).all() and torch.isnan(c.lse[2]).all()
        c.check(rows=None if fits else {0, 1})


@pytest.mark.parametrize("nope,rope", [(448, 64), (64, 16)])
def test_rows_of_no_slot_are_left_out(cuda, nope, rope):
    c = Case(cuda, [(4, 90), (3, 40), (6, 200)], 32, page=16, nope=nope, rope=rope, seed=47)
    c.q_start.copy_(torch.tensor([2, 4, 7, 11]))       # rows 0, 1, 11 and 12 belong to nobody
    c.starts = np.array([2, 4, 7, 11])
    c.seqs = [(2, 90), (3, 40), (4, 200)]
    c.run()
    c.check()
    for r in (0, 1, 11, 12):
        assert (c.out[r] == 77).all() and (c.lse[r] == 77).all()


@pytest.mark.parametrize("nope,rope", [(448, 64), (64, 16)])
def test_tokens_before_the_first_position(cuda, nope, rope):
    """More new tokens than positions: the first of them see nothing."""
    c = Case(cuda, [(5, 90), (1, 30)], 16, page=16, nope=nope, rope=rope, seed=53)
    c.use_sink = False
    c.pool.length[0] = 3                               # tokens at -2 .. 2
    c.run()
    torch.cuda.synchronize()
    assert (c.out[:2] == 0).all() and torch.isneginf(c.lse[:2]).all()
    c.seqs[0] = (5, 3)
    c.check(rows={2, 3, 4, 5})


@pytest.mark.parametrize("nope,rope,heads", [(64, 16, 1), (448, 64, 130), (512, 128, 5),
                                             (512, 512, 17), (64, 2, 40), (64, 0, 9)])
@pytest.mark.parametrize("seqs", [((1, 1),), ((1, 31), (1, 33)), ((1, 1500),),
                                  ((40, 100), (0, 5), (3, 300))])
def test_general_shapes_and_lengths(cuda, nope, rope, heads, seqs):
    """One token to many, keys in one piece and in several, heads that do not
    fill their blocks, rows without RoPE values."""
    c = Case(cuda, list(seqs), heads, page=48, nope=nope, rope=rope, seed=nope + heads)
    c.use_rope = rope > 0
    c.run()
    c.check()
    a, b = c.out.clone(), c.lse.clone()
    c.run()
    assert torch.equal(a, c.out) and torch.equal(b, c.lse)


def test_general_shapes_with_windows_and_holes(cuda):
    c = Case(cuda, [(30, 300), (1, 700), (2, 2)], 20, page=16, window=130, nope=128, rope=32,
             freed=True, seed=59)
    c.table[1, 38:41] = -1
    c.pool.table.copy_(torch.from_numpy(c.table).int())
    c.run()
    c.check()


def test_odd_rows_are_refused(cuda):
    cache = cuda.LatentCache.from_tensors(
        torch.zeros(64, 64, dtype=torch.uint8, device="cuda"),
        torch.zeros(64, 8, dtype=torch.uint8, device="cuda"),
        torch.zeros(64, 3, dtype=torch.int16, device="cuda"))
    pool = cuda.PagedCache.empty([cache], 16, 2, 4)
    q = torch.zeros(1, 4, 67, device="cuda")
    with pytest.raises(cuda.Dsv4CudaError, match="odd"):
        cuda.paged_attn(torch.empty_like(q), q, pool, 0,
                        torch.zeros(3, dtype=torch.int32, device="cuda"), 1, 16, 1.0)


@pytest.mark.parametrize("nope,rope", [(448, 64), (64, 16)])
def test_every_slot_beyond(cuda, nope, rope):
    c = Case(cuda, [(3, 100), (1, 700)], 16, page=16, nope=nope, rope=rope, seed=61)
    cuda.paged_attn(c.out, c.q, c.pool, 0, c.q_start, 0, 700, c.scale, lse=c.lse)
    assert c.pool.status() == 4
    assert torch.isnan(c.out).all() and torch.isnan(c.lse).all()
