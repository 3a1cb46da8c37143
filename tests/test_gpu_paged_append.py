"""dsv4cuda_paged_append where its rows are longer or shorter than the new tokens: a
captured step has rows for the most tokens that it may bring. Whole numbers, compared
exactly."""
import pytest
import torch

pytestmark = pytest.mark.gpu

PAGE = 4


def pool_of(cuda, pages=16, seqs=4, width=4):
    return cuda.PagedCache.empty([cuda.LatentCache(pages * PAGE, 64, 2)], PAGE, seqs, width)


def dev(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


def rows_of(n):
    return torch.full((n,), 3, dtype=torch.int64, device="cuda")


def test_rows_behind_the_tokens_are_none(cuda):
    """3 is a live row here: written there, a step's padding would overwrite it."""
    pool = pool_of(cuda)
    rows = rows_of(700)
    pool.append(dev([0, 2]), dev([5, 1]), rows)
    assert rows.tolist() == [0, 1, 2, 3, 4, 8] + [-1] * 694
    rows = rows_of(5)
    pool.append(dev([0, 2]), dev([0, 0]), rows)
    assert rows.tolist() == [-1] * 5
    rows = rows_of(5)
    pool.append(dev([]), dev([]), rows)
    assert rows.tolist() == [-1] * 5
    assert pool.length.tolist() == [5, 0, 1, 0] and pool.status() == 0


def test_a_captured_step_brings_fewer_tokens_than_before(cuda):
    pool = pool_of(cuda)
    slots, counts, rows = dev([0, 1]), dev([3, 2]), rows_of(6)
    pool.append(slots, counts, rows)            # (the first call sets the kernels up)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        pool.append(slots, counts, rows)
    for n0, n1, want in ((2, 3, [3, 8, 6, 7, 12, -1]), (1, 0, [9, -1, -1, -1, -1, -1]),
                         (0, 2, [13, 14, -1, -1, -1, -1])):
        counts.copy_(dev([n0, n1]))
        g.replay()
        assert rows.tolist() == want
    assert pool.status() == 0


def test_tokens_beyond_the_rows_are_refused(cuda):
    """An op whose tokens have no room in rows changes nothing."""
    pool = pool_of(cuda)
    pool.append(dev([0]), dev([6]))
    rows = rows_of(8)
    pool.append(dev([0, 1, 2, 3]), dev([3, 4, 2, 0]), rows)     # 9 tokens, the last 2 too many
    assert rows.tolist() == [6, 7, 8, 12, 13, 14, 15, -1]
    assert pool.length.tolist() == [9, 4, 0, 0]
    assert pool.table.tolist() == [[0, 1, 2, -1], [3, -1, -1, -1], [-1] * 4, [-1] * 4]
    assert pool.refs.tolist() == [1] * 4 + [0] * 12
    assert pool.status() == pool.BAD_OP
    # an op that is left out for another reason has its place in rows all the same
    rows = rows_of(4)
    pool.append(dev([2, 9, 3]), dev([1, 2, 2]), rows)
    assert rows.tolist() == [16, -1, -1, -1]
    assert pool.length.tolist() == [9, 4, 1, 0] and pool.status() == pool.BAD_OP
    pool.append(dev([3]), dev([1]), torch.empty(0, dtype=torch.int64, device="cuda"))
    assert pool.length.tolist() == [9, 4, 1, 0] and pool.status() == pool.BAD_OP
    pool.append(dev([3]), dev([1]))                             # no rows wanted: no limit
    assert pool.length.tolist() == [9, 4, 1, 1] and pool.status() == 0


def test_nobody_overtakes_an_op_without_pages(cuda):
    """4 pages, 1 of them taken: the second op needs 4, the third one that there is, the
    last none."""
    pool = pool_of(cuda, pages=4)
    pool.append(dev([3]), dev([2]))
    rows = rows_of(25)
    pool.append(dev([0, 1, 2, 3]), dev([4, 16, 3, 2]), rows)
    assert rows.tolist() == [4, 5, 6, 7] + [-1] * 19 + [2, 3]
    assert pool.length.tolist() == [4, 0, 0, 4]
    assert pool.refs.tolist() == [1, 1, 0, 0] and pool.status() == pool.EXHAUSTED
