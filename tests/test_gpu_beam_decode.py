"""Beams of prompts decoded as a server would: norm to 8 bits, latents appended, written and attended
to, the residual's norm, routed experts of two kinds of routes, a head of grouped products, selection
and fork. Each operator is held to 64 bits on the inputs that it got (bounds of its own tests, and of
test_gpu_paged_attn's attention), the totals to their steps' logits, the pages to every beam's own
ancestors; the same steps captured once and replayed give the same bits."""
import pytest
import torch

import grouped_ref as ref
import test_gpu_beam as beam_ref
import test_gpu_moe_experts as moe_ref

pytestmark = pytest.mark.gpu
G, B, CANDS, HIDDEN, HEADS, VOCAB, PAGE, STEPS, LEN = 3, 4, 8, 512, 64, 1003, 4, 7, 12
N, DIM, ROPE = G * B, 512, 64
EPS = 2.0 ** -19
LAST = ("tok", "score", "slot", "pos")


class Decoder:
    def __init__(self, cuda, seed=0):
        self.cuda = cuda
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)

        def w(*shape):
            return (torch.randn(*shape, device="cuda", generator=g) * shape[-1] ** -0.5).bfloat16()

        def gain(n):
            return (1 + 0.1 * torch.randn(n, device="cuda", generator=g)).bfloat16()
        self.embed, self.gains = w(VOCAB, HIDDEN) * 8, [gain(HIDDEN) for _ in range(3)]
        self.wq, self.wkv = w(HEADS * DIM, HIDDEN), w(DIM, HIDDEN)
        self.wo, self.gate = w(HIDDEN, HEADS * DIM), w(16, HIDDEN)
        self.gain_kv, self.sink = gain(DIM), torch.randn(HEADS, device="cuda", generator=g)
        self.layer, self.weights = moe_ref.layer_of(cuda, HIDDEN, 256, 16, 3, seed=seed)
        self.head, self.head_scale = ref.fp8(1, VOCAB, HIDDEN, g)
        self.cache = cuda.LatentCache((LEN // PAGE + 1) * N * PAGE)
        self.pool = cuda.PagedCache.empty([self.cache], PAGE, N, LEN // PAGE)
        self.freq = 1e4 ** (-torch.arange(0, ROPE, 2, device="cuda") / ROPE)
        i32 = dict(dtype=torch.int32, device="cuda")
        self.start, self.ones = torch.arange(N + 1, **i32), torch.ones(N, **i32)
        self.offsets = torch.tensor([0, N], **i32)
        self.tok = torch.arange(N, device="cuda") * 7 % VOCAB
        self.score = torch.full((G, B), -float("inf"), device="cuda")
        self.score[:, 0] = 0  # a prompt starts as one beam
        self.slot = torch.randperm(N, device="cuda", generator=g).int().view(G, B)
        self.pos = torch.zeros(N, dtype=torch.int64, device="cuda")
        f32, u8 = dict(dtype=torch.float32, device="cuda"), dict(dtype=torch.uint8, device="cuda")
        self.rows = torch.empty(N, dtype=torch.int64, device="cuda")
        for name in ("codes", "codes2", "codes3"):
            setattr(self, name, torch.empty(N, HIDDEN, **u8))
            setattr(self, name.replace("codes", "scales"), torch.empty(N, HIDDEN // 128, **u8))
        for name in ("y", "h", "hn", "m"):
            setattr(self, name, torch.empty(N, HIDDEN, dtype=torch.bfloat16, device="cuda"))
        self.o = torch.empty(N, HEADS, DIM, dtype=torch.bfloat16, device="cuda")
        self.new = torch.empty(N, DIM, **f32)
        self.logits = torch.empty(N, VOCAB, **f32)
        self.parent, self.token = torch.empty(G, CANDS, **i32), torch.empty(G, CANDS, **i32)
        self.total = torch.empty(G, CANDS, **f32)
        self.next, self.dst, self.src = (torch.empty(G, B, **i32) for _ in range(3))
        need = max(self.layer.experts_workspace_bytes(N),
                   cuda.grouped_workspace_bytes(self.logits, self.codes3, self.head, N))
        self.work = torch.empty(need, **u8)
        probe = torch.empty(N, HEADS, DIM, dtype=torch.bfloat16, device="cuda")
        self.attn_work = torch.empty(cuda.paged_attn_workspace_bytes(probe, self.pool, 1, LEN), **u8)

    def step(self):
        """Tokens tok of the beams, one each, to the next ones; every tensor stays where it is."""
        c = self.cuda
        self.x = self.embed[self.tok]
        c.norm_quant(self.x, self.gains[0], self.codes, self.scales, out=self.y)
        flat = self.slot.flatten()
        order = torch.argsort(flat)
        a = self.pos[:, None].float() * self.freq
        self.cos, self.sin = a.cos(), a.sin()
        self.q, self.kv = (self.y @ self.wq.T).view(N, HEADS, DIM), self.y @ self.wkv.T
        self.pool.append(flat, self.ones, self.rows)
        self.pool.write(0, self.kv, self.rows, self.gain_kv, rope_cos=self.cos, rope_sin=self.sin)
        self.cache.read(self.rows, self.new)  # (the fork below may hand on the page)
        o = torch.empty_like(self.o)
        c.paged_attn(o, self.q[order], self.pool, 0, self.start, 1, LEN, DIM ** -0.5, sink=self.sink,
                     workspace=self.attn_work)
        self.o[order] = o
        self.r = self.o.flatten(1) @ self.wo.T
        c.norm_quant(self.x, self.gains[1], self.codes2, self.scales2, residual=self.r,
                     sum_out=self.h, out=self.hn)
        p = torch.sigmoid(self.hn @ self.gate.T).float()
        wt, idx = p.topk(3, dim=1)
        self.idx, at = idx.int().sort(dim=1)
        self.wt = wt.gather(1, at).contiguous()
        self.layer.experts(self.codes2, self.scales2, self.idx, self.wt, self.m, workspace=self.work)
        c.norm_quant(self.h, self.gains[2], self.codes3, self.scales3, residual=self.m)
        c.grouped_gemm(self.logits, self.codes3, self.scales3, self.head, self.head_scale, self.offsets,
                       workspace=self.work)
        self.was = self.slot.clone(), self.score.clone()
        c.beam_select(self.logits, self.score, self.parent, self.token, self.total, self.next,
                      slot=self.slot, dst=self.dst, src=self.src, eos=5)
        self.pool.fork(self.dst.flatten(), self.src.flatten())
        on = self.next.long()
        alive, on = on >= 0, on.clamp(min=0)
        self.tok.copy_(self.token.gather(1, on).clamp(min=0).flatten())
        self.score.copy_(torch.where(alive, self.total.gather(1, on), -float("inf")))
        self.mother = torch.where(alive, self.parent.gather(1, on), -1)
        self.slot.copy_(self.dst)
        # an emptied slot starts over
        self.pos.copy_(self.pool.length[self.slot.flatten().long()].long())

    def result(self):
        return [getattr(self, n).clone() for n in LAST] + [
            self.logits.clone(), self.pool.table.clone(), self.pool.refs.clone(), self.pool.length.clone(),
            self.cache.codes.clone(), self.cache.scales.clone(), self.cache.rope.clone()]


def normed(v, gain, eps=1e-6):
    return v / torch.sqrt((v * v).mean(dim=1, keepdim=True) + eps) * gain.double()


def check_codes(codes, scales, y):
    low, high = ref.quantised_range(y, EPS * y.abs())
    got = ref.rows_of(codes, scales)
    assert bool(((got >= low) & (got <= high)).all())


def check_step(d, history):
    """The last step's operators in 64 bits; history: each beam's latents, with the step's own."""
    v = normed(d.x.double(), d.gains[0])
    check_codes(d.codes, d.scales, v)
    assert bool(((d.y.double() - v).abs() <= (2.0 ** -8 + 2 * EPS) * v.abs()).all())
    # attention over what the pages hold: a beam's own ancestors
    for b in range(N):
        k = torch.stack(history[b]).double()
        q = d.q[b].double()
        s = q @ k.T * DIM ** -0.5
        p = torch.softmax(torch.cat([s, d.sink.double()[:, None]], 1), 1)[:, :-1]
        dx = 2 * 2.0 ** -24 * DIM * DIM ** -0.5 * float((q.abs() @ k.abs().T).max())
        bound = (2.0 ** -8 + 4 * dx + 2.0 ** -11) * (p @ k.abs())
        assert bool(((d.o[b].double() - p @ k).abs() <= bound).all())
    v = d.x.double() + d.r.double()
    check_codes(d.codes2, d.scales2, normed(v, d.gains[1]))
    assert bool(((d.h.double() - v).abs() <= 2.0 ** -8 * (1 + 2.0 ** -15) * v.abs()).all())
    y, bound = moe_ref.want(d.weights, d.codes2, d.scales2, d.idx, d.wt)
    assert bool(((d.m.double() - y).abs() <= bound).all())
    check_codes(d.codes3, d.scales3, normed(d.h.double() + d.m.double(), d.gains[2]))
    x, w = ref.rows_of(d.codes3, d.scales3), ref.fp8_of(d.head, d.head_scale)[0]
    y = x @ w.T
    assert bool(((d.logits.double() - y).abs() <= ref.sum_bound(x, w) + 2.0 ** -23 * y.abs()).all())
    slot, score = d.was
    t = beam_ref.check(d.cuda, d.logits, score, CANDS, eos=5, slot=slot)
    for a, b in zip(t, (d.parent, d.token, d.total, d.next, d.dst, d.src)):
        assert torch.equal(a, b.cpu())


def test_steps_and_their_replay(cuda):
    d = Decoder(cuda)
    history = [[] for _ in range(N)]  # a beam's latents as the cache holds them
    forks = 0
    for _ in range(STEPS):
        pos = d.pos.clone()
        d.step()
        new = d.new
        for b in range(N):
            assert len(history[b]) == int(pos[b])
            history[b] = history[b] + [new[b].clone()]
        # the write, within its bounds
        v = normed(d.kv.double(), d.gain_kv)
        low, high = ref.quantised_range(v[:, :448], EPS * v[:, :448].abs(), 64)
        assert bool(((new[:, :448] >= low) & (new[:, :448] <= high)).all())
        a, b = v[:, 448::2], v[:, 449::2]
        c, s = d.cos.double(), d.sin.double()
        turned = torch.stack([a * c - b * s, a * s + b * c], 2).flatten(1)
        size = (a.abs() + b.abs()).repeat_interleave(2, dim=1)
        assert bool(((new[:, 448:] - turned).abs() <= 2.0 ** -8 * turned.abs() + 2 * EPS * size).all())
        check_step(d, history)
        mother = d.mother.tolist()
        forks += sum(m.count(b) > 1 for m in mother for b in range(B))
        history = [history[g * B + m] if m >= 0 else [] for g in range(G) for m in mother[g]]
        # the pages hold every beam's ancestors
        for b, s in enumerate(d.slot.flatten().tolist()):
            n = int(d.pool.length[s])
            assert n == len(history[b])
            if n:
                t = torch.arange(n, device="cuda")
                rows = d.pool.table[s].long()[t // PAGE] * PAGE + t % PAGE
                got = torch.empty(n, DIM, device="cuda")
                d.cache.read(rows, got)
                assert torch.equal(got, torch.stack(history[b]))
        held = torch.bincount(d.pool.table[d.pool.table >= 0].long(), minlength=d.pool.n_pages)
        assert torch.equal(held.int(), d.pool.refs)
    assert d.pool.status() == 0 and cuda.device_error() == 0
    assert forks >= G
    eager = d.result()
    d.layer.close()

    d = Decoder(cuda)  # one step as it is, the others replayed
    d.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        d.step()
    for _ in range(STEPS - 1):
        graph.replay()
    for a, b in zip(eager, d.result()):
        assert torch.equal(a, b)
    assert d.pool.status() == 0 and cuda.device_error() == 0
    del graph
    d.layer.close()
