"""Rows of long tiles whose softmax one key dominates, against 64 bits.

The weights of P V are BF16 in tiles of more than a few key blocks, and the running
maximum moves only when a score exceeds it by 8 (log2 units), so the dominating key's
weight is any number up to 2^8 and rounds like any other. Every product of a score but
one is zero here, so the scores are exact.

Tolerance. With u = 2^-8 a weight is held as w_t (1 + d_t), |d_t| <= u. The sums are
divided by the sum of the weights as they are held, the sink's share left as it is, so
    got = sum p_t (1 + d_t - d) v_t,  d = sum p_t d_t / sum p_t,
and since sum p_t (d_t - d) = 0 the error sum p_t (d_t - d) v_t equals
sum p_t (d_t - d) (v_t - c) for every c. With c = the mean of v under the weights alone
(o without the sink) it is sum p_t d_t (v_t - c): at most u sum p_t |v_t - c|. The
output's rounding adds u |o| (|got| itself at most (1 + u) times that). What is left is
fp32: a weight's exponent, at most 8 in size, is off by 2^-23 of itself in the product
and as much in the factor, exp2 by 2^-22, the sums of at most 1024 weights in partial
sums of 64 by 2^-18: below 2^-16 of A = sum p_t |v_t| together. So
    |got - want| <= u (sum p_t |v_t - c| + (1 + u) |o|) + 2^-16 A,
    |lse - want| <= 2^-16 (1 + |want|).
Where a key with a weight near one has all of the row, that is the output's rounding
alone. (A tile that is cut into parts has each part's O divided by the part's own sum:
the same with c the part's mean. Two keys hold all of a row's weight here, so c is their
mean, or the key itself.)"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

HEADS, NOPE, ROPE, PAGE = 64, 448, 64, 64
U = 2.0 ** -8


def build(cuda, seqs, low, high, bf16, seed):
    """Slots of (new, length); position `low` has score 0, `high` the head's factor, the
    others -64 times it: RoPE value 0 is the only one that the queries look at."""
    rng = np.random.default_rng(seed)
    held = [-(-length // PAGE) for _, length in seqs]
    rows = sum(held) * PAGE
    codes = torch.from_numpy((rng.normal(size=(rows, NOPE)) * 100).astype(np.float32))
    codes = codes.clamp(-448, 448).to(torch.float8_e4m3fn)
    scales = torch.from_numpy(rng.integers(117, 123, (rows, 8)).astype(np.uint8))
    rope = torch.from_numpy(rng.normal(size=(rows, ROPE)).astype(np.float32)).bfloat16()
    order = rng.permutation(sum(held))
    table = np.full((len(seqs), max(held)), -1)
    at = 0
    for s, h in enumerate(held):
        table[s, :h] = order[at:at + h]
        at += h
        for t in range(h * PAGE):
            rope[table[s, t // PAGE] * PAGE + t % PAGE, 0] = \
                0.0 if t == low else 1.0 if t == high else -64.0
    value = codes.double().view(rows, NOPE // 64, 64) * (
        2.0 ** (scales[:, :NOPE // 64].double() - 127))[:, :, None]
    value = torch.cat([value.flatten(1), rope.double()], 1).numpy()
    cache = cuda.LatentCache.from_tensors(codes.view(torch.uint8).cuda(), scales.cuda(),
                                          rope.cuda().view(torch.int16))
    i32 = dict(dtype=torch.int32, device="cuda")
    pool = cuda.PagedCache([cache], PAGE, torch.tensor(table, **i32),
                           torch.tensor([b for _, b in seqs], **i32),
                           torch.ones(sum(held), **i32))
    total = sum(n for n, _ in seqs)
    factor = torch.from_numpy(rng.uniform(1.0, 5.5, (total, HEADS)).astype(np.float32)).bfloat16()
    q = torch.zeros(total, HEADS, NOPE + ROPE, dtype=torch.bfloat16)
    q[:, :, NOPE] = factor
    q = q.to(torch.bfloat16 if bf16 else torch.float32).cuda()
    return pool, table, value, q


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("use_sink", [False, True])
@pytest.mark.parametrize("seqs,low,high,window", [
    (((1, 1000),), 520, 590, 0),                # cut into several shares and merged
    (((400, 1000),), 520, 590, 0),              # tiles inside a share, tiles cut by one
    (((400, 1000),), 520, 590, 500),            # blocks that the window cuts
    (((70, 300), (1, 700), (3, 500)), 100, 170, 0)])
def test_a_dominating_key(cuda, seqs, low, high, window, use_sink, bf16):
    pool, table, value, q = build(cuda, seqs, low, high, bf16, seed=len(seqs) * 7 + window)
    total = q.shape[0]
    out, lse = torch.empty_like(q), torch.empty(total, HEADS, device="cuda")
    starts = np.concatenate([[0], np.cumsum([n for n, _ in seqs])])
    sink = np.linspace(-1.0, 1.0, HEADS).astype(np.float32)
    cuda.paged_attn(out, q, pool, 0, torch.tensor(starts, dtype=torch.int32, device="cuda"),
                    max(n for n, _ in seqs), max(b for _, b in seqs), 1.0,
                    sink=torch.from_numpy(sink).cuda() if use_sink else None, window=window,
                    lse=lse)
    torch.cuda.synchronize()
    got, got_lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    qd = q.double().cpu().numpy()
    for s, (n, length) in enumerate(seqs):
        for i in sorted({0, 1, n // 3, n // 2, n - 2, n - 1} & set(range(n))):
            r, pos = starts[s] + i, length - n + i
            t = np.arange(max(0, pos - window + 1) if window else 0, pos + 1)
            assert low in t and high in t
            v = value[table[s, t // PAGE] * PAGE + t % PAGE]
            x = qd[r] @ v.T
            full = np.concatenate([x, sink.astype(np.float64)[:, None]], 1) if use_sink else x
            m = full.max(1, keepdims=True)
            e = np.exp(full - m)
            den = e.sum(1, keepdims=True)
            p = (e / den)[:, :len(t)]
            want = p @ v
            mean = want / p.sum(1, keepdims=True)
            around = np.einsum("hk,hkd->hd", p, np.abs(v[None] - mean[:, None]))
            tol = U * (around + (1 + U) * np.abs(want)) + 2.0 ** -16 * (p @ np.abs(v)) + 1e-30
            assert (np.abs(got[r] - want) <= tol).all(), (s, i, (np.abs(got[r] - want) / tol).max())
            want_lse = (m + np.log(den))[:, 0]
            assert (np.abs(got_lse[r] - want_lse) <= 2.0 ** -16 * (1 + np.abs(want_lse))).all()
    assert pool.status() == 0
