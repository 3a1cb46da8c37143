"""Pages of the latent cache (dsv4cuda_paged_append / _fork / _compact) against
a model of the tables in plain Python. Everything here is whole numbers and
copied bytes, so every comparison is exact."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


class Model:
    """The tables as lists, the op rules as loops."""

    def __init__(self, pages, page, seqs, width):
        self.page, self.width = page, width
        self.table = [[-1] * width for _ in range(seqs)]
        self.length = [0] * seqs
        self.refs = [0] * pages
        self.status = 0
        # what each cache row holds, as a tag: (layer-independent) number or None
        self.held = [None] * (pages * page)

    def free_pages(self):
        return [q for q, r in enumerate(self.refs) if r == 0]

    def fork(self, dst, src):
        n, seqs = len(dst), len(self.table)
        owner = {}
        for i, d in enumerate(dst):
            if 0 <= d < seqs:
                owner.setdefault(d, i)
        ops = []
        for i, (d, s) in enumerate(zip(dst, src)):
            ok = 0 <= d < seqs and -1 <= s < seqs and owner[d] == i
            if ok and s >= 0 and s != d and s in owner and src[owner[s]] != s:
                ok = False
            if not ok:
                self.status |= 2
            elif s != d:
                ops.append((d, s))
        for d, _ in ops:
            for q in self.table[d]:
                if q >= 0:
                    self.refs[q] -= 1
            self.table[d] = [-1] * self.width
        free = self.free_pages()
        todo, used = [], 0
        for d, s in ops:
            part = s >= 0 and self.length[s] % self.page and \
                self.table[s][self.length[s] // self.page] >= 0
            if part:
                page = free[used] if used < len(free) else None
                used += 1
                todo.append((d, s, page, True))
            else:
                todo.append((d, s, None, False))
        moves = []
        for d, s, page, part in todo:
            if s < 0 or (part and page is None):
                self.length[d] = 0
                self.status |= 1 if s >= 0 else 0
                continue
            full, rest = divmod(self.length[s], self.page)
            for j in range(full):
                q = self.table[s][j]
                self.table[d][j] = q
                if q >= 0:
                    self.refs[q] += 1
            if part:
                self.table[d][full] = page
                self.refs[page] = 1
                a, b = self.table[s][full] * self.page, page * self.page
                moves.append((a, b, rest))
            self.length[d] = self.length[s]
        old = list(self.held)
        for a, b, k in moves:
            self.held[b:b + k] = old[a:a + k]

    def append(self, slots, counts, n_rows):
        free = self.free_pages()
        used, seen, rows = 0, set(), []
        for s, c in zip(slots, counts):
            ok = 0 <= s < len(self.table) and c >= 0 and s not in seen
            if 0 <= s < len(self.table):
                seen.add(s)
            if ok:
                L = self.length[s]
                ok = L + c <= self.width * self.page
                if ok and c > 0 and L % self.page:
                    q = self.table[s][L // self.page]
                    ok = q >= 0 and self.refs[q] == 1
            if not ok:
                self.status |= 2
                rows += [-1] * max(c, 0)
                continue
            have, want = -(-L // self.page), -(-(L + c) // self.page)
            first = used
            used += want - have
            if want > have and used > len(free):
                self.status |= 1
                rows += [-1] * c
                continue
            for j in range(want - have):
                self.table[s][have + j] = free[first + j]
                self.refs[free[first + j]] = 1
            for p in range(L, L + c):
                rows.append(self.table[s][p // self.page] * self.page + p % self.page)
            self.length[s] = L + c
        if len(rows) > n_rows:
            self.status |= 2
        return rows[:n_rows]

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        holes = [q for q in range(live) if self.refs[q] == 0]
        moves = [q for q in range(live, len(self.refs)) if self.refs[q] > 0]
        to = dict(zip(moves, holes))
        for q, t in to.items():
            self.refs[t], self.refs[q] = self.refs[q], 0
            P = self.page
            self.held[t * P:t * P + P] = self.held[q * P:q * P + P]
        self.table = [[to.get(q, q) for q in row] for row in self.table]


def make(cuda, layers, pages, page, seqs, width, nope=448, rope=64):
    caches = [cuda.LatentCache(pages * page + 3, nope, rope) for _ in range(layers)]
    pool = cuda.PagedCache.empty(caches, page, seqs, width)
    if pool.n_pages != pages:  # the rows behind the last whole page make none
        pool = cuda.PagedCache(caches, page, pool.table, pool.length,
                               torch.zeros(pages, dtype=torch.int32, device="cuda"))
    return pool


def dev(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


def stamp(pool, rows, tags):
    """Writes tag-dependent bytes into cache rows, another pattern per layer."""
    for layer, c in enumerate(pool.caches):
        for r, t in zip(rows, tags):
            if r >= 0:
                c.codes[r] = (t * 7 + layer) % 120
                c.scales[r] = (t + layer) % 200
                c.rope[r] = t + layer


def check(pool, model):
    torch.cuda.synchronize()
    assert pool.table.cpu().tolist() == model.table
    assert pool.length.cpu().tolist() == model.length
    assert pool.refs.cpu().tolist() == model.refs
    for layer, c in enumerate(pool.caches):
        codes, scales, rope = (t.cpu().numpy() for t in (c.codes, c.scales, c.rope))
        for s, row in enumerate(model.table):
            for p in range(model.length[s]):
                q = row[p // model.page]
                if q < 0:
                    continue
                r = q * model.page + p % model.page
                t = model.held[r]
                if t is None:
                    continue
                assert (codes[r] == (t * 7 + layer) % 120).all(), (s, p)
                assert (scales[r] == (t + layer) % 200).all()
                assert (rope[r] == t + layer).all()


@pytest.mark.parametrize("layers,pages,page,seqs,width,nope,rope", [
    (1, 40, 16, 6, 9, 448, 64), (3, 23, 7, 9, 6, 64, 16), (2, 9, 1, 5, 8, 448, 64),
    (2, 64, 33, 12, 5, 128, 10), (64, 12, 4, 4, 6, 64, 2)])
def test_random_ops_follow_the_model(cuda, layers, pages, page, seqs, width, nope, rope):
    rng = np.random.default_rng(pages * 31 + page)
    pool = make(cuda, layers, pages, page, seqs, width, nope, rope)
    model = Model(pages, page, seqs, width)
    tag = 0
    for step in range(14):
        kind = ["append", "append", "fork", "compact", "fork", "append"][step % 6]
        if kind == "append":
            n = int(rng.integers(1, seqs + 1))
            slots = rng.permutation(seqs)[:n].tolist()
            counts = rng.integers(0, page * 3 + 2, n).tolist()
            total = sum(counts)
            rows = torch.full((max(total, 1),), -7, dtype=torch.int64, device="cuda")
            pool.append(dev(slots), dev(counts), rows)
            want = model.append(slots, counts, max(total, 1))
            torch.cuda.synchronize()
            got = rows.cpu().tolist()[:total]
            assert got == want
            tags = list(range(tag, tag + total))
            tag += total
            stamp(pool, got, tags)
            for r, t in zip(got, tags):
                if r >= 0:
                    model.held[r] = t
        elif kind == "fork":
            half = max(1, seqs // 2)
            dst = rng.permutation(np.arange(half, seqs))[:int(rng.integers(1, seqs - half + 1))]
            src = rng.integers(-1, half, dst.size)
            pool.fork(dev(dst.tolist()), dev(src.tolist()))
            model.fork(dst.tolist(), src.tolist())
        else:
            pool.compact()
            model.compact()
        check(pool, model)
    assert pool.status() == model.status


def test_ops_that_cannot_be_done(cuda):
    pool = make(cuda, 1, 8, 4, 6, 3)
    model = Model(8, 4, 6, 3)

    def both(name, a, b, n_rows=64):
        if name == "append":
            rows = torch.full((n_rows,), -7, dtype=torch.int64, device="cuda")
            pool.append(dev(a), dev(b), rows)
            want = model.append(a, b, n_rows)
            torch.cuda.synchronize()
            assert rows.cpu().tolist()[:len(want)] == want
            for r in want:
                if r >= 0:
                    model.held[r] = None
        else:
            pool.fork(dev(a), dev(b))
            model.fork(a, b)
        check(pool, model)
        assert pool.status() == model.status
        model.status = 0

    both("append", [0, 1, 0, -1, 9], [6, 5, 2, 3, 1])       # named twice, out of range
    both("append", [2], [13])                               # more than the table holds
    both("append", [2, 3], [-1, 0])                         # negative; nothing
    both("append", [2, 3], [12, 8])                         # the second finds no pages
    both("fork", [4, 4, 7, 5], [0, 1, 0, -2])               # named twice, out of range
    both("fork", [4, 5, 0], [0, 4, -1])                     # 5 <- 4 is replaced by 4 <- 0
    both("fork", [1, 3], [1, 1])                            # 1 stays, 3 copies it
    both("append", [0, 1, 2, 3, 4, 5], [1, 1, 1, 1, 1, 1])
    both("fork", [5, 4, 3], [2, 1, 2])                      # sharing only, or no page left
    both("append", [1, 3], [9, 4], n_rows=3)                # rows shorter than the tokens
    both("fork", [0, 1, 2, 3, 4, 5], [-1] * 6)
    assert pool.refs.sum().item() == 0


def test_append_behind_a_shared_partial_page(cuda):
    pool = make(cuda, 1, 8, 4, 2, 3)
    pool.append(dev([0]), dev([6]))
    pool.table[1] = pool.table[0]                           # as fork would not leave it
    pool.length[1] = 6
    pool.refs[:2] += 1
    rows = torch.zeros(2, dtype=torch.int64, device="cuda")
    pool.append(dev([1]), dev([2]), rows)
    assert rows.tolist() == [-1, -1]
    assert pool.length.tolist() == [6, 6]
    assert pool.status() == pool.BAD_OP


def test_pages_given_back_inside_a_sequence(cuda):
    """A window's server frees pages from the front (-1 entries): they are
    neither shared nor counted."""
    pool = make(cuda, 1, 10, 4, 3, 5)
    pool.append(dev([0]), dev([15]))
    pool.table[0, :2] = -1
    pool.refs[:2] = 0
    pool.fork(dev([1]), dev([0]))
    assert pool.table.tolist()[1] == [-1, -1, 2, 0, -1]
    assert pool.refs.tolist() == [1, 0, 2, 1] + [0] * 6
    assert pool.length.tolist() == [15, 15, 0]


def test_compact_into_other_tables(cuda):
    """The old tables stay valid for the steps that still read them."""
    pool = make(cuda, 2, 30, 8, 6, 6)
    pool.append(dev([0, 1, 2, 3, 4, 5]), dev([20, 33, 9, 40, 17, 24]))
    for c in pool.caches:
        c.codes.random_(0, 100)
        c.rope.random_(0, 1000)
    pool.free(dev([0, 2, 3]))
    before = [(c.codes.clone(), c.rope.clone()) for c in pool.caches]
    t0, r0 = pool.table.clone(), pool.refs.clone()
    t1, r1 = torch.empty_like(t0), torch.empty_like(r0)
    pool.compact(t1, r1)
    assert torch.equal(pool.table, t0) and torch.equal(pool.refs, r0)
    live = int((r0 > 0).sum())
    assert (r1[:live] > 0).all() and (r1[live:] == 0).all()
    for s in (1, 4, 5):
        pos = torch.arange(int(pool.length[s]), device="cuda")
        old = t0[s][pos // 8].long() * 8 + pos % 8
        new = t1[s][pos // 8].long() * 8 + pos % 8
        for c, (codes, rope) in zip(pool.caches, before):
            assert torch.equal(c.codes[new], codes[old]) and torch.equal(c.codes[old], codes[old])
            assert torch.equal(c.rope[new], rope[old])


@pytest.mark.parametrize("pages", [1, 1023, 1024, 5000, 40000])
def test_large_pools(cuda, pages):
    """Free pages far apart in a pool of more pages than a block has threads."""
    rng = np.random.default_rng(pages)
    cache = cuda.LatentCache(pages, 64, 2)
    seqs, width = 40, 700
    pool = cuda.PagedCache.empty([cache], 1, seqs, width)
    model = Model(pages, 1, seqs, width)
    refs = (rng.random(pages) < 0.97).astype(np.int32)      # held by somebody else
    pool.refs.copy_(torch.from_numpy(refs))
    model.refs = refs.tolist()
    slots = rng.permutation(seqs).tolist()
    counts = rng.integers(0, 60, seqs).tolist()
    rows = torch.zeros(sum(counts), dtype=torch.int64, device="cuda")
    pool.append(dev(slots), dev(counts), rows)
    assert rows.tolist() == model.append(slots, counts, sum(counts))
    assert pool.table.tolist() == model.table and pool.refs.tolist() == model.refs
    assert pool.status() == model.status
    pool.compact()
    model.held = [None] * pages
    model.compact()
    assert pool.refs.tolist() == model.refs and pool.table.tolist() == model.table


def test_captured_and_on_another_stream(cuda):
    pool = make(cuda, 1, 16, 4, 4, 4)
    slots, counts = dev([0, 1]), dev([1, 2])
    rows = torch.zeros(3, dtype=torch.int64, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pool.append(slots, counts, rows)
    torch.cuda.current_stream().wait_stream(side)
    assert rows.tolist() == [0, 4, 5]
    three, one = dev([3]), dev([1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        pool.append(slots, counts, rows)
        pool.fork(three, one)
    model = Model(16, 4, 4, 4)
    model.append([0, 1], [1, 2], 3)
    for _ in range(4):
        g.replay()
        want = model.append([0, 1], [1, 2], 3)
        model.fork([3], [1])
        assert rows.tolist() == want
        assert pool.table.tolist() == model.table and pool.refs.tolist() == model.refs


def test_refusals(cuda):
    pool = make(cuda, 1, 8, 4, 3, 3)
    i32 = dict(dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        pool.fork(torch.zeros(1, dtype=torch.int64, device="cuda"), torch.zeros(1, **i32))
    with pytest.raises(ValueError):
        pool.fork(torch.zeros(2, **i32), torch.zeros(1, **i32))
    with pytest.raises(ValueError):
        pool.append(torch.zeros(1, **i32), torch.zeros(1, **i32), torch.zeros(4, **i32))
    with pytest.raises(ValueError):
        pool.compact(torch.zeros(3, 2, **i32))
    with pytest.raises(ValueError):
        pool.append(torch.zeros(2, 2, **i32)[:, 0], torch.zeros(2, **i32))
    with pytest.raises(cuda.Dsv4CudaError, match="one op per slot"):
        pool.fork(torch.zeros(4, **i32), torch.zeros(4, **i32))
    small = cuda.LatentCache(31)
    with pytest.raises(cuda.Dsv4CudaError, match="fewer than 32 rows"):
        cuda.PagedCache([small], 4, pool.table, pool.length, pool.refs).compact()
    other = cuda.LatentCache(32, 64, 16)
    with pytest.raises(cuda.Dsv4CudaError, match="cache 1"):
        cuda.PagedCache([cuda.LatentCache(32), other], 4, pool.table, pool.length,
                        pool.refs).compact()
    with pytest.raises(cuda.Dsv4CudaError):
        cuda.PagedCache([small] * 65, 3, pool.table, pool.length, pool.refs).compact()
    short = cuda.PagedCache(pool.caches, 4, pool.table, pool.length, pool.refs)
    short.struct.workspace_bytes = 8
    with pytest.raises(cuda.Dsv4CudaError, match="workspace"):
        short.compact()
