"""Arguments of paged_attn that are refused before anything is launched: what they would
have the kernels read or write is not theirs."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture
def call(cuda):
    """paged_attn of two tokens of one slot; a keyword replaces its argument."""
    pool = cuda.PagedCache.empty([cuda.LatentCache(64)], 16, 1, 4)
    pool.append(torch.zeros(1, dtype=torch.int32, device="cuda"),
                torch.full([1], 30, dtype=torch.int32, device="cuda"))
    for t in (pool.caches[0].codes, pool.caches[0].rope):
        t.zero_()
    pool.caches[0].scales.fill_(127)
    q = torch.ones(2, 8, 512, dtype=torch.bfloat16, device="cuda")
    out = torch.full_like(q, 5.0)
    q_start = torch.tensor([0, 2], dtype=torch.int32, device="cuda")

    def f(q=q, out=out, **kw):
        cuda.paged_attn(out, q, pool, 0, q_start, 2, 30, 1.0, **kw)
        return out
    return f


def test_expanded_rows(call):
    one = torch.ones(1, 8, 512, dtype=torch.bfloat16, device="cuda")
    for kw in (dict(q=one.expand(2, 8, 512)), dict(out=one.expand(2, 8, 512))):
        with pytest.raises(ValueError, match="overlap"):
            call(**kw)
    assert (one == 1).all()
    assert (call() == 0).all()                  # still usable


def test_a_workspace_that_is_none(call):
    for ws in (torch.empty(1 << 24, dtype=torch.uint8),
               torch.empty(1 << 22, dtype=torch.float32, device="cuda"),
               torch.empty(1 << 25, dtype=torch.uint8, device="cuda")[::2]):
        with pytest.raises(ValueError, match="workspace"):
            call(workspace=ws)
    assert (call(workspace=torch.empty(1 << 24, dtype=torch.uint8, device="cuda")) == 0).all()
