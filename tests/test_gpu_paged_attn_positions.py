"""paged_attn where a difference of positions could leave the range of an int: the widest
windows, lengths below the new tokens' number, lengths that are none."""
import pytest
import torch

pytestmark = pytest.mark.gpu

WIDEST = 2 ** 31 - 1


@pytest.mark.parametrize("nope,rope", [(448, 64), (64, 16)])
@pytest.mark.parametrize("window", [WIDEST, WIDEST - 1, WIDEST - 40, 701])
@pytest.mark.parametrize("lengths", [(3, 90, 700), (0, 1, 700), (-1, -40, 600),
                                     (-WIDEST - 1, -WIDEST, 64)])
def test_a_window_beyond_every_length_is_none(cuda, nope, rope, window, lengths):
    """The same bits as without a window; tokens at positions below 0 see nothing."""
    tokens, page, pages = (5, 40, 3), 16, 60
    g = torch.Generator(device="cuda").manual_seed(7)

    def ints(lo, hi, *shape, dtype):
        return torch.randint(lo, hi, shape, device="cuda", generator=g, dtype=dtype)
    cache = cuda.LatentCache.from_tensors(ints(0, 120, pages * page, nope, dtype=torch.uint8),
                                          ints(117, 123, pages * page, 8, dtype=torch.uint8),
                                          torch.randn(pages * page, rope, device="cuda", generator=g)
                                          .bfloat16().view(torch.int16))
    i32 = dict(dtype=torch.int32, device="cuda")
    table = torch.full((3, 50), -1, **i32)
    table[0, :1], table[1, :6], table[2, :44] = 50, torch.arange(44, 50, **i32), \
        torch.arange(44, **i32)
    pool = cuda.PagedCache([cache], page, table, torch.tensor(lengths, **i32),
                           torch.zeros(pages, **i32))
    total, heads, dim = sum(tokens), 8, nope + rope
    q = torch.randn(total, heads, dim, device="cuda", generator=g).bfloat16()
    q_start = torch.tensor([0, 5, 45, 48], **i32)
    got = []
    for w in (0, window):
        out = torch.full_like(q, 77.0)
        lse = torch.full((total, heads), 77.0, device="cuda")
        cuda.paged_attn(out, q, pool, 0, q_start, 40, 700, dim ** -0.5, window=w, lse=lse)
        got.append((out, lse))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    out, lse = got[1]
    row = 0
    for n, length in zip(tokens, lengths):
        blind = n - max(0, min(n, length))
        assert (out[row:row + blind] == 0).all() and torch.isneginf(lse[row:row + blind]).all()
        assert torch.isfinite(out[row + blind:row + n]).all()
        assert torch.isfinite(lse[row + blind:row + n]).all()
        row += n
    assert pool.status() == 0
