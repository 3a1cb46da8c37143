"""Prompts served from one pool of latent pages: admitted, read in chunks, scored,
forked into samples, decoded token by token, released and compacted.

    python examples/serve_prompts.py

One attention layer of random weights stands for a model's: what matters is the
order of the calls. Every call is asynchronous on the current stream and depends on
device memory alone, so a server can capture a step of them in a graph.
"""
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "deepseek-v4-flash-0731-in-c_b200"))
import dsv4cuda as d4  # noqa: E402

HEADS, DIM, ROPE, HIDDEN, VOCAB, PAGE = 64, 512, 64, 256, 4099, 16
SLOTS = 12


class Layer:
    """Random projections of a hidden row to queries and a latent, and a vocabulary head."""

    def __init__(self, seed):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)

        def w(*shape):
            return torch.randn(*shape, device="cuda", generator=g) * shape[-1] ** -0.5
        self.embed = torch.randn(VOCAB, HIDDEN, device="cuda", generator=g)
        self.wq, self.wkv = w(HEADS * DIM, HIDDEN), w(DIM, HIDDEN)
        self.wo, self.head = w(HIDDEN, HEADS * DIM), w(VOCAB, HIDDEN)
        self.sink = torch.randn(HEADS, device="cuda", generator=g)
        self.freq = 10000.0 ** (-torch.arange(0, ROPE, 2, device="cuda") / ROPE)

    def rope(self, x, pos, sign=1.0):
        a = pos[:, None].float() * self.freq[None]
        c, s = a.cos(), a.sin() * sign
        while c.dim() < x.dim():
            c, s = c.unsqueeze(1), s.unsqueeze(1)
        x = x.clone()
        u, v = x[..., -ROPE::2].clone(), x[..., 1 - ROPE::2].clone()
        x[..., -ROPE::2], x[..., 1 - ROPE::2] = u * c - v * s, u * s + v * c
        return x

    def step(self, server, slots, tokens, counts, pos):
        """tokens (all slots', one behind the other) at positions pos: their latents go to
        the pool, each attends to its sequence, and the logits come out."""
        x = self.embed[tokens]
        q = self.rope((x @ self.wq.T).view(-1, HEADS, DIM), pos).bfloat16()
        kv = self.rope(x @ self.wkv.T, pos).bfloat16().float()
        rows = torch.empty(len(tokens), dtype=torch.int64, device="cuda")
        server.pool.append(slots, counts, rows)
        server.cache.write(kv, rows)
        # each slot's rows of q: its new tokens, none for the others
        new = torch.zeros(SLOTS, dtype=torch.int32, device="cuda")
        new[slots.long()] = counts
        order = torch.argsort(torch.repeat_interleave(slots, counts), stable=True)
        q_start = torch.zeros(SLOTS + 1, dtype=torch.int32, device="cuda")
        q_start[1:] = new.cumsum(0)
        a = pos[order][:, None].float() * self.freq[None]
        out = torch.empty_like(q)
        d4.paged_attn(out, q[order], server.pool, 0, q_start, int(counts.max()), server.max_len,
                      DIM ** -0.5, sink=self.sink, rope_cos=a.cos().contiguous(),
                      rope_sin=a.sin().contiguous())
        back = torch.empty_like(out)
        back[order] = out
        return (back.float().flatten(1) @ self.wo.T + x) @ self.head.T


class Server:
    def __init__(self, pages=64, max_len=160):
        self.cache = d4.LatentCache(pages * PAGE)
        self.pool = d4.PagedCache.empty([self.cache], PAGE, SLOTS, -(-max_len // PAGE))
        self.max_len = max_len


def score(logits, tokens, top=4):
    n = len(tokens)
    f32, i32 = dict(dtype=torch.float32, device="cuda"), dict(dtype=torch.int32, device="cuda")
    got = dict(logprob=torch.empty(n, **f32), entropy=torch.empty(n, **f32),
               rank=torch.empty(n, **i32), top_id=torch.empty(n, top, **i32),
               top_logprob=torch.empty(n, top, **f32))
    d4.token_logprobs(logits, tokens, **got)
    return got


def serve(seed=0, samples=3, steps=6, prompts=(37, 70), chunk=32):
    """Returns the server, the layer, each slot's tokens and their log probabilities."""
    layer, server = Layer(seed), Server()
    g = torch.Generator().manual_seed(seed)
    texts, logprobs = {}, {}
    last = {}
    for s, n in enumerate(prompts):  # a prompt's chunks, one after another
        text = torch.randint(0, VOCAB, (n,), generator=g).cuda()
        texts[s], logprobs[s] = text.tolist(), []
        for at in range(0, n, chunk):
            part = text[at:at + chunk]
            logits = layer.step(server, torch.tensor([s], dtype=torch.int32, device="cuda"), part,
                                torch.tensor([len(part)], dtype=torch.int32, device="cuda"),
                                torch.arange(at, at + len(part), device="cuda"))
            # each token scored by the logits before it; the last one's follower is not known
            follow = torch.full((len(part),), -1, dtype=torch.int32, device="cuda")
            known = text[at + 1:at + 1 + len(part)]
            follow[:len(known)] = known.int()
            logprobs[s] += score(logits, follow)["logprob"][:len(known)].tolist()
        last[s] = logits[-1]
    # samples share their prompt's full pages
    dst = list(range(len(prompts), len(prompts) * (1 + samples)))
    src = [i % len(prompts) for i in range(len(dst))]
    server.pool.fork(torch.tensor(dst, dtype=torch.int32, device="cuda"),
                     torch.tensor(src, dtype=torch.int32, device="cuda"))
    slots = torch.tensor(dst, dtype=torch.int32, device="cuda")
    ones = torch.ones_like(slots)
    logits = torch.stack([last[s] for s in src])
    for s, d in zip(src, dst):
        texts[d], logprobs[d] = list(texts[s]), list(logprobs[s])
    for _ in range(steps):
        alternatives = score(logits, torch.full_like(slots, -1), top=samples)
        # sample i takes the i-th alternative, so that the samples part
        pick = torch.arange(len(dst), device="cuda") // len(prompts)
        tokens = alternatives["top_id"].gather(1, pick[:, None])[:, 0]
        chosen = score(logits, tokens)
        for i, d in enumerate(dst):
            logprobs[d].append(chosen["logprob"][i].item())
            texts[d].append(int(tokens[i]))
        pos = server.pool.length[slots.long()].long()
        logits = layer.step(server, slots, tokens.long(), ones, pos)
    # the prompts' own slots and one sample are done; the rest closes ranks
    gone = [*range(len(prompts)), dst[0]]
    server.pool.free(torch.tensor(gone, dtype=torch.int32, device="cuda"))
    server.pool.compact()
    if server.pool.status():
        raise RuntimeError("an operation on the pool could not be done")
    for s in gone:
        del texts[s], logprobs[s]
    return server, layer, texts, logprobs


if __name__ == "__main__":
    server, layer, texts, logprobs = serve()
    used = int((server.pool.refs > 0).sum())
    print(f"{len(texts)} samples left in {used} of {server.pool.n_pages} pages")
    for s, text in texts.items():
        print(f"slot {s}: {len(text)} tokens, mean log probability "
              f"{sum(logprobs[s]) / len(logprobs[s]):.3f}")
