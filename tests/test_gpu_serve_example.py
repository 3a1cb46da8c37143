"""examples/serve_prompts.py: prompts in chunks, forks, decode steps, release and
compaction through one pool, against each sequence computed alone in 64 bits.

Tolerance: a log probability follows the logits, which are linear in the attention's
outputs (BF16: 2^-8 of their value sums, as tests/test_gpu_paged_attn.py derives) and
in latents that the reference rounds to the cache's grid in fp32 here and there alike.
The head is fp32 with weights of size HIDDEN^-1/2, so a logit's error is about 2^-8 /
sqrt(keys) of an output of size about 1 and a log probability's about twice that:
0.02 covers a single key and all roundings after it; the mean over a sequence is an
order smaller."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location(
        "serve_prompts", os.path.join(ROOT, "examples", "serve_prompts.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def plain_logprobs(m, server, layer, slot, text):
    """The sequence alone, from the latents that the pool holds for it."""
    n = len(text)
    pos = torch.arange(n, device="cuda")
    page = server.pool.table[slot].long()[pos // m.PAGE]
    assert (page >= 0).all()
    rows = page * m.PAGE + pos % m.PAGE
    k = torch.empty(n, m.DIM, device="cuda")
    server.cache.read(rows, k)
    k = k.double()
    x = layer.embed[torch.tensor(text, device="cuda")]
    q = layer.rope((x @ layer.wq.T).view(-1, m.HEADS, m.DIM), pos).bfloat16().double()
    s = torch.einsum("nhd,kd->hnk", q, k) * m.DIM ** -0.5
    s = s.masked_fill(pos[None, None, :] > pos[None, :, None], float("-inf"))
    s = torch.cat([s, layer.sink.double()[:, None, None].expand(-1, n, 1)], 2)
    o = torch.einsum("hnk,kd->nhd", torch.softmax(s, 2)[..., :-1], k)
    o = layer.rope(o, pos, -1.0).flatten(1)
    logits = (o @ layer.wo.double().T + x.double()) @ layer.head.double().T
    lp = torch.log_softmax(logits, 1)
    return lp[:-1].gather(1, torch.tensor(text[1:], device="cuda")[:, None])[:, 0]


@pytest.mark.parametrize("seed,prompts,chunk", [(0, (37, 70), 32), (1, (16, 1, 48), 7)])
def test_samples_of_shared_prompts(cuda, example, seed, prompts, chunk):
    server, layer, texts, logprobs = example.serve(seed=seed, prompts=prompts, chunk=chunk)
    assert len(texts) == 3 * len(prompts) - 1
    used = int((server.pool.refs > 0).sum())
    assert (server.pool.refs[:used] > 0).all()
    held = torch.bincount(server.pool.table[server.pool.table >= 0].long(),
                          minlength=server.pool.n_pages)
    assert torch.equal(held.int(), server.pool.refs)
    for slot, text in texts.items():
        got = torch.tensor(logprobs[slot], device="cuda", dtype=torch.float64)
        want = plain_logprobs(example, server, layer, slot, text)
        assert got.shape == want.shape
        assert (got - want).abs().max().item() < 0.02
        assert (got - want).mean().abs().item() < 0.005
