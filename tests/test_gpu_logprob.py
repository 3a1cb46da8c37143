"""dsv4cuda_token_logprobs against 64-bit log softmax.

Tolerances. Z is a sum of V positive fp32 terms, at most V / 128 of them one
after another in a thread and the rest in a tree, each term exp(x - m) with
the argument rounded to 24 bits and the exponential to about 2 ulp: its
relative error, and so log Z's absolute one, is below
E = 2^-24 (V / 128 + 16 + 2 D), D the largest finite m - x that counts (a
term below e^-25 / V adds less than 2^-24 in all, so D <= 25 + log V). A log
probability adds two roundings of its own size. The entropy's sum carries the
same relative error on every term e^d |d|, of total S = sum p |d|, and the
division another E: E (2 + 2 S) + 2^-22 (log Z + S)."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
V = 129280


def run(cuda, x, tokens, top, stream=None):
    n = x.shape[0]
    f32 = dict(dtype=torch.float32, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    lp, en = torch.full((n,), 9e9, **f32), torch.full((n,), 9e9, **f32)
    rank = torch.full((n,), -9, **i32)
    ti, tl = torch.full((n, top), -9, **i32), torch.full((n, top), 9e9, **f32)
    cuda.token_logprobs(x, tokens, lp, en, rank, ti if top else None, tl if top else None,
                        stream=stream)
    return lp, en, rank, ti, tl


def check(cuda, x, tokens, top, stream=None):
    lp, en, rank, ti, tl = run(cuda, x, tokens, top, stream)
    torch.cuda.synchronize()
    n, vocab = x.shape
    y = x.double().cpu().numpy()
    t = tokens.cpu().numpy()
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        m = y.max(axis=1)
        ref = np.where(np.isneginf(m), 0.0, m)
        d = y - ref[:, None]
        e = np.exp(d)
        z = e.sum(axis=1)
        lz = np.where(np.isneginf(m), 0.0, np.log(np.where(z > 0, z, 1)))
        S = np.where(e > 0, e * -d, 0.0).sum(axis=1) / np.where(z > 0, z, 1)
    E = 2.0 ** -24 * (vocab / 128 + 16 + 2 * (25 + math.log(vocab)))
    broken = np.isnan(y).any(axis=1) | np.isposinf(m)
    for r in range(n):
        asked = 0 <= t[r] < vocab
        order = np.lexsort((np.arange(vocab), -y[r]))
        order = order[~np.isnan(y[r][order])]
        ids = np.full(top, -1)
        ids[:min(top, order.size)] = order[:top]
        assert ti[r].cpu().numpy().tolist() == ids.tolist(), r
        got = tl[r].cpu().numpy().astype(np.float64)
        if not asked:
            assert lp[r].item() == 0.0 and rank[r].item() == -1
        if broken[r]:
            assert math.isnan(en[r].item()) and np.isnan(got).all()
            assert not asked or math.isnan(lp[r].item())
            continue
        if asked:
            xt = y[r, t[r]]
            assert rank[r].item() == int((y[r] > xt).sum() + (y[r, :t[r]] == xt).sum())
            want = xt - ref[r] - lz[r]
            if math.isinf(want):
                assert lp[r].item() == want
            else:
                assert abs(lp[r].item() - want) <= E + 2.0 ** -22 * (abs(xt) + abs(ref[r]) + lz[r])
        wt = y[r, ids[ids >= 0]] - ref[r] - lz[r]
        got = got[ids >= 0]
        inf = np.isinf(wt)
        assert np.array_equal(got[inf], wt[inf])
        assert np.all(np.abs(got[~inf] - wt[~inf])
                      <= E + 2.0 ** -22 * (np.abs(wt[~inf]) + 2 * abs(ref[r]) + lz[r]))
        want = 0.0 if np.isneginf(m[r]) else lz[r] + S[r]
        assert abs(en[r].item() - want) <= E * (2 + 2 * S[r]) + 2.0 ** -22 * (lz[r] + S[r])


def rows(rng, n, vocab, dtype, pad=0, scale=2.5):
    x = torch.from_numpy((rng.normal(size=(n, vocab + pad)) * scale).astype(np.float32))
    x = x.to(dtype).cuda()
    x[:, vocab:] = 1e30
    return x[:, :vocab]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,vocab,pad,top", [
    (1, 1, 0, 1), (3, 2, 5, 2), (1, 31, 0, 31), (2, 33, 1, 32), (5, 1000, 3, 0), (7, 4097, 0, 20),
    (1, V, 0, 20), (6, V, 37, 5), (40, 32000, 1, 32), (300, 517, 0, 8), (1, 1000003, 0, 32)])
def test_sizes(cuda, dtype, n, vocab, pad, top):
    rng = np.random.default_rng(n * 7 + vocab)
    x = rows(rng, n, vocab, dtype, pad)
    t = torch.from_numpy(rng.integers(0, vocab, n).astype(np.int32)).cuda()
    check(cuda, x, t, top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [64, 777, 50000])
def test_masks_ties_and_broken_rows(cuda, dtype, vocab):
    rng = np.random.default_rng(vocab)
    x = rows(rng, 16, vocab, dtype)
    lowest = torch.finfo(dtype).min
    x[0] = -math.inf                                  # nothing left
    x[1] = -math.inf
    x[1, vocab // 2] = 3.0                            # one left
    x[2] = lowest                                     # a mask of the type's lowest value
    x[3] = lowest
    x[3, 5:9] = 1.0
    x[4] = 0.0
    x[4, ::2] = -0.0                                  # equal values of either sign
    x[5, 7] = math.nan
    x[6, 9] = math.inf
    x[7] = math.nan
    x[8] = torch.arange(vocab, device="cuda").to(dtype) * 0.01    # ascending: the worst order
    x[9] = -torch.arange(vocab, device="cuda").to(dtype) * 0.01
    x[10, torch.rand(vocab, device="cuda") < 0.97] = -math.inf
    x[11] = 1e30 if dtype is torch.float32 else 2.0 ** 60
    x[11, 3] = -x[11, 0]
    x[12] = -1e30
    x[13] = (torch.arange(vocab, device="cuda") % 3).to(dtype)    # many ties
    t = torch.arange(16, device="cuda", dtype=torch.int32) * 3 % vocab
    t[14], t[15] = -1, vocab
    check(cuda, x, t, min(32, vocab))


@pytest.mark.parametrize("n,vocab", [(1, V), (2, 70001), (200, 9001)])
def test_order_does_not_matter(cuda, n, vocab):
    """Ascending rows make every element a candidate; results stay the definition's,
    and a second run gives the same bits."""
    x = torch.arange(vocab, device="cuda").float()[None].repeat(n, 1) * 1e-4
    t = torch.full((n,), vocab // 3, dtype=torch.int32, device="cuda")
    check(cuda, x, t, 32)
    a, b = run(cuda, x, t, 32), run(cuda, x, t, 32)
    assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_on_another_stream_and_captured(cuda):
    rng = np.random.default_rng(1)
    x = rows(rng, 4, 5000, torch.float32)
    t = torch.tensor([1, 2, 3, 4], dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        check(cuda, x, t, 4)
    lp = torch.zeros(4, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cuda.token_logprobs(x, t, lp)
    x.mul_(0.5)
    g.replay()
    want = torch.log_softmax(x.double(), 1).gather(1, t[:, None].long())[:, 0]
    assert (lp.double() - want).abs().max().item() < 1e-5


def test_rows_beyond_32_bit_offsets(cuda):
    """Rows whose element offsets pass 2^31."""
    vocab, n = 200_000, 11_000
    x = torch.zeros(n, vocab, dtype=torch.bfloat16, device="cuda")
    x[-1, 77] = 5.0
    x[-1, 12345] = 4.0
    t = torch.zeros(n, dtype=torch.int32, device="cuda")
    t[-1] = 12345
    lp, en, rank, ti, tl = run(cuda, x, t, 2)
    assert ti[-1].tolist() == [77, 12345] and rank[-1].item() == 1
    assert ti[0].tolist() == [0, 1] and rank[0].item() == 0
    assert abs(lp[0].item() + math.log(vocab)) < 1e-4
    want = 4.0 - math.log(vocab - 2 + math.exp(5) + math.exp(4))
    assert abs(lp[-1].item() - want) < 1e-4


def test_refusals(cuda):
    x = torch.zeros(2, 10, device="cuda")
    t = torch.zeros(2, dtype=torch.int32, device="cuda")
    lp = torch.zeros(2, device="cuda")

    def top(k):
        return (torch.zeros(2, k, dtype=torch.int32, device="cuda"),
                torch.zeros(2, k, device="cuda"))
    with pytest.raises(cuda.Dsv4CudaError):
        cuda.token_logprobs(x, t, lp, None, None, *top(11))       # more than the vocabulary
    with pytest.raises(cuda.Dsv4CudaError):
        cuda.token_logprobs(torch.zeros(2, 99, device="cuda"), t, lp, None, None, *top(33))
    with pytest.raises(cuda.Dsv4CudaError):
        cuda.token_logprobs(torch.zeros(2, 0, device="cuda"), t, lp)
    with pytest.raises(ValueError):
        cuda.token_logprobs(x, t.long(), lp)
    with pytest.raises(ValueError):
        cuda.token_logprobs(x.half(), t, lp)
    with pytest.raises(ValueError):
        cuda.token_logprobs(x.t(), t, lp)
    with pytest.raises(ValueError):
        cuda.token_logprobs(x, t[:1], lp)
    with pytest.raises(ValueError):
        cuda.token_logprobs(x, t, lp, None, None, top(3)[0], torch.zeros(2, 2, device="cuda"))
    cuda.token_logprobs(x[:0], t[:0], lp[:0])                      # no rows: nothing to do


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,vocab,pad", [(1, V, 0), (48, V, 37), (700, 20011, 0), (9, 1260, 3),
                                         (1500, 1260, 0), (5, 300, 1)])
@pytest.mark.parametrize("top", [1, 5, 32])
def test_few_values_left(cuda, dtype, n, vocab, pad, top):
    """Masks that leave less than the alternatives asked for: what is masked fills
    up by its index, NaN among the first values does not."""
    rng = np.random.default_rng(vocab + top)
    x = rows(rng, n, vocab, dtype, pad)
    for r in range(n):
        left = [0, 1, top - 1, top, top + 1, 40][r % 6]
        keep = torch.from_numpy(rng.choice(vocab, left, replace=False)).cuda()
        values = x[r, keep].clone()
        x[r] = -math.inf
        if r % 5 == 3:
            x[r, :250] = math.nan
        x[r, keep] = values
    t = torch.from_numpy(rng.integers(0, vocab, n).astype(np.int32)).cuda()
    check(cuda, x, t, top)
