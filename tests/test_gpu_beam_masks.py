"""dsv4cuda_beam_select where logits are masked by large finite values, against 64-bit log softmax
(test_gpu_beam.check). A term is e^(v - ref) of a difference rounded to 24 bits, scaled by log2 e with
a second rounding and the constant's own 2^-26: |v - ref| (2.2) 2^-24 of itself, 55 2^-24 at 25
(beyond, terms add nothing), 17 2^-24 for the additions and 4 2^-24 for the exponential: below the
2^-17 that check allows. v - ref is exact at v = ref whatever its size."""
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
