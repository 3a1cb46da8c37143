"""Reference counts that do not fit the tables: a pool built over pages that a caller never
counted. Their release leaves counts below zero, and what follows stays inside the pool."""
import pytest
import torch

pytestmark = pytest.mark.gpu

PAGE = 4


def dev(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


def pool_of(cuda, table, length, refs):
    cache = cuda.LatentCache(len(refs) * PAGE, 64, 2)
    row = torch.arange(len(refs) * PAGE, device="cuda")
    cache.codes.copy_((row[:, None] % 100).expand(-1, 64))
    return cuda.PagedCache([cache], PAGE, dev(table), dev(length), dev(refs))


def test_compact_after_pages_without_a_count_were_given_back(cuda):
    # slot 0 holds pages 1, 4, 5 that nobody counted; slot 1 holds 7 and 9, counted
    pool = pool_of(cuda, [[1, 4, 5], [7, 9, -1]], [12, 7], [0] * 7 + [1, 0, 1, 0, 0])
    pool.free(dev([0]))
    assert pool.refs.tolist() == [0, -1, 0, 0, -1, -1, 0, 1, 0, 1, 0, 0]
    pool.compact()
    assert pool.table.tolist() == [[-1] * 3, [0, 1, -1]]
    assert pool.refs.tolist() == [1, 1, 0, 0, -1, -1] + [0] * 6
    codes = pool.caches[0].codes[:, 0].tolist()
    assert codes[0:4] == [28, 29, 30, 31] and codes[4:8] == [36, 37, 38, 39]
    assert codes[8:] == list(range(8, 48))          # nothing else was written
    assert pool.status() == 0


def test_pages_below_zero_are_taken(cuda):
    pool = pool_of(cuda, [[-1] * 3] * 2, [0, 0], [-1, 1, -2, 0, -5])
    rows = torch.zeros(11, dtype=torch.int64, device="cuda")
    pool.append(dev([1, 0]), dev([9, 2]), rows)
    assert rows.tolist() == [0, 1, 2, 3, 8, 9, 10, 11, 12, 16, 17]
    assert pool.refs.tolist() == [1] * 5 and pool.status() == 0


def test_compact_of_any_counts(cuda):
    g = torch.Generator().manual_seed(3)
    for n in (1, 3, 64, 5000):
        refs = torch.randint(-2, 3, (n,), generator=g).tolist()
        pool = pool_of(cuda, [[-1]], [0], refs)
        pool.compact()
        live = sum(r > 0 for r in refs)
        holes = [q for q in range(live) if refs[q] <= 0]
        moves = [q for q in range(live, n) if refs[q] > 0]
        for a, b in zip(moves, holes):
            refs[b], refs[a] = refs[a], 0
        assert pool.refs.tolist() == refs
