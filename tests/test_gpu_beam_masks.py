"""dsv4cuda_beam_select where logits are masked by large finite values, or are large themselves,
against 64-bit log softmax (test_gpu_beam.check). A term is e^(v - ref) of a difference rounded to 24
bits, scaled by log2 e with a second rounding and the constant's own 2^-26: |v - ref| (2.2) 2^-24 of
itself, 55 2^-24 at 25 (beyond, terms add nothing), 17 2^-24 for the additions and 4 2^-24 for the
exponential: below the 2^-17 that check allows. v - ref is exact at v = ref whatever its size."""
import pytest
import torch

from test_gpu_beam import check

pytestmark = pytest.mark.gpu
MASKS = ["lowest", -1e30, -1e20, -1e10, -1e9]


def value(mask, dtype):
    return torch.finfo(dtype).min if mask == "lowest" else mask


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("groups,beams,vocab,cands", [
    (1, 3, 90, 5), (1, 4, 129280, 8), (12, 3, 9000, 6), (12, 2, 129280, 4), (10, 8, 33000, 16)])
def test_few_live_logits(cuda, dtype, mask, groups, beams, vocab, cands):
    """All but a few logits are masked, so that most threads see none: the live ones come first, the
    lowest masked tokens after them."""
    g = generator(vocab + groups)
    x = torch.full((groups * beams, vocab), value(mask, dtype), device="cuda")
    for r in range(groups * beams):
        at = torch.randperm(vocab, device="cuda", generator=g)[:1 + r % 7]
        x[r, at] = torch.randn(len(at), device="cuda", generator=g) * 3
    score = -torch.arange(1, beams + 1, device="cuda").float().repeat(groups, 1) * 0.75
    slot = torch.arange(groups * beams, dtype=torch.int32, device="cuda").view(groups, beams)
    parent, token, total, *_ = check(cuda, x.to(dtype), score, cands, slot=slot)
    assert bool((parent[:, 0] >= 0).all()) and bool((total[:, 0] > -100).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("level", MASKS + [1e9, 1e10, 1e20, 1e30, -5.3e10, 5.3e10, "largest"])
@pytest.mark.parametrize("groups,vocab", [(1, 77), (1, 129280), (11, 20000)])
def test_rows_of_one_value(cuda, dtype, level, groups, vocab):
    """Uniform, whatever the value: each token's total is the score less log vocab."""
    v = torch.finfo(dtype).max if level == "largest" else value(level, dtype)
    x = torch.full((groups * 2, vocab), v, device="cuda").to(dtype)
    score = torch.tensor([[-1.0, -2.0]], device="cuda").repeat(groups, 1)
    parent, token, total, *_ = check(cuda, x, score, 8)
    assert token.tolist() == [list(range(8))] * groups
    assert bool((parent == 0).all())
    want = -1 - torch.tensor(float(vocab), dtype=torch.float64).log()
    assert bool(((total.double() - want).abs() <= 2.0 ** -17 + 2.0 ** -24 * want.abs()).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("top", [1e9, 1e20, 1e30])
@pytest.mark.parametrize("groups", [1, 11])
def test_large_logits(cuda, dtype, top, groups):
    """Rows with one large logit, early or late, and rows that climb or fall through many powers: every
    thread's sum is moved, most of them to nothing."""
    vocab = 40000
    g = generator(groups)
    x = torch.randn(groups * 4, vocab, device="cuda", generator=g)
    x[0::4, 3] = top
    x[1::4, vocab - 5] = top
    steps = torch.linspace(0, 1, vocab, device="cuda")
    x[2::4] = top ** steps
    x[3::4] = -(top ** steps)
    score = -torch.arange(1, 5, device="cuda").float().repeat(groups, 1)
    check(cuda, x.to(dtype), score, 12)


def test_large_and_lowest_together(cuda):
    """A first step of the lowest values, then ordinary ones, then the largest; and a row with an
    infinity or NaN behind masked values, which has no continuations still."""
    low, high = torch.finfo(torch.float32).min, 1e30
    x = torch.full((24, 60000), low, device="cuda")
    x[:, 30000:45000] = torch.randn(24, 15000, device="cuda", generator=generator(5))
    x[0::3, 59000] = high
    x[4, 50], x[7, 59999] = float("inf"), float("nan")
    score = -torch.arange(1, 4, device="cuda").float().repeat(8, 1)
    parent, *_ = check(cuda, x, score, 7)
    assert not bool((parent[1] == 1).any()) and not bool((parent[2] == 1).any())
