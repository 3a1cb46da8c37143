"""dsv4cuda_moe_experts against 64 bits. Bound: gate and up carry grouped_ref's error of a sum;
through the gate function (slope at most 1.1) and the products with up and weight that moves h by
eps (and 2^-20 of it, the roundings of exponential and division); h is rounded to E4M3, so it may
come out anywhere between the roundings of h - eps and h + eps; a slot adds its sum's error and
half a BF16 step, the token's sum another."""
import pytest
import torch

import grouped_ref as ref

pytestmark = pytest.mark.gpu


def layer_of(cuda, hidden, inter, experts, topk, limit=10, seed=0, part=None):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    lo, hi = part or (0, experts)
    w = dict(hidden=hidden, moe_inter=inter, n_experts=experts, topk=topk, swiglu_limit=limit,
             route_scale=1.5, gate_w=torch.zeros(experts, hidden, dtype=torch.int16, device="cuda"))
    for a, outs, width in ((1, inter, hidden), (3, inter, hidden), (2, hidden, inter)):
        q, s = ref.fp4(experts, outs, width, g)
        w[f"w{a}"], w[f"s{a}"] = q[lo:hi].contiguous(), s[lo:hi].contiguous()
    return cuda.MoeLayer(w, max_tokens=1, device=True, expert_range=part), w


def routes(n, experts, topk, seed=1):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    idx = torch.rand(n, experts, device="cuda", generator=g).topk(topk, dim=1).indices
    return idx.sort(dim=1).values.int(), torch.rand(n, topk, device="cuda", generator=g) + 0.05


def want(w, xq, xs, idx, wt, lo=0):
    x = ref.rows_of(xq, xs)
    out = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(out)
    L = float(w["swiglu_limit"])
    for e in range(w["w1"].shape[0]):
        t, k = (idx == e + lo).nonzero(as_tuple=True)
        if not len(t):
            continue
        m1, m3, m2 = (ref.fp4_of(w[f"w{a}"][e], w[f"s{a}"][e]) for a in (1, 3, 2))
        g, u = x[t] @ m1.T, x[t] @ m3.T
        eg, eu = ref.sum_bound(x[t], m1), ref.sum_bound(x[t], m3)
        g, u = g.clamp(max=L), u.clamp(-L, L)
        r = wt[t, k].double()[:, None]
        h = g * torch.sigmoid(g) * u * r
        eps = r * (1.1 * eg * (u.abs() + eu) + (g * torch.sigmoid(g)).abs() * eu) + 2.0 ** -20 * h.abs()
        q, _ = ref.quantised(h)
        low, high = ref.quantised_range(h, eps)
        slack = torch.maximum(high - q, q - low)
        y = q @ m2.T
        b = ref.sum_bound(q.abs() + slack, m2) + slack @ m2.abs().T
        b = b + 2.0 ** -8 * (y.abs() + b)
        out.index_add_(0, t, y)
        bound.index_add_(0, t, b)
    return out, bound + 2.0 ** -8 * (out.abs() + bound)


def check(cuda, layer, w, xq, xs, idx, wt, lo=0):
    out = torch.full(xq.shape, 7.0, dtype=torch.bfloat16, device="cuda")
    layer.experts(xq, xs, idx, wt, out)
    y, b = want(w, xq, xs, idx, wt, lo)
    d = (out.double() - y).abs()
    assert bool((d <= b + 1e-30).all()), float((d / (b + 1e-30)).max())
    # rows that come out far inside the bound, so that it hides no wrong row
    assert float(d.norm()) <= 0.01 * float(y.norm()) + 1e-30
    again = torch.empty_like(out)
    layer.experts(xq, xs, idx, wt, again)
    assert torch.equal(out, again)
    assert cuda.device_error() == 0
    return out


CASES = [  # n, hidden, inter, experts, topk
    (1, 256, 128, 16, 2), (1, 4096, 2048, 8, 6), (7, 128, 256, 3, 3), (33, 384, 128, 4, 1),
    (100, 640, 384, 40, 8), (600, 512, 256, 5, 2), (1500, 256, 128, 64, 6), (2, 7168, 256, 256, 8),
]


# either product may have the longer sums, the wider rows and so the larger tiles
UNEVEN = [(1500, 128, 4096, 2, 2), (600, 7168, 128, 2, 2), (5000, 128, 3584, 3, 2), (3000, 3584, 128, 4, 1)]


@pytest.mark.parametrize("n,hidden,inter,experts,topk", UNEVEN)
def test_uneven(cuda, n, hidden, inter, experts, topk):
    layer, w = layer_of(cuda, hidden, inter, experts, topk)
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    xq, xs = ref.activations(n, hidden, g)
    idx, wt = routes(n, experts, topk)
    need = layer.experts_workspace_bytes(n)
    room = torch.full((need + 65536,), 0x5A, dtype=torch.uint8, device="cuda")
    out = check(cuda, layer, w, xq, xs, idx, wt)
    again = torch.empty_like(out)
    layer.experts(xq, xs, idx, wt, again, workspace=room[:need])
    assert torch.equal(out, again) and bool((room[need:] == 0x5A).all())
    layer.close()


@pytest.mark.parametrize("n,hidden,inter,experts,topk", CASES)
def test_experts(cuda, n, hidden, inter, experts, topk):
    layer, w = layer_of(cuda, hidden, inter, experts, topk)
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    xq, xs = ref.activations(n, hidden, g)
    idx, wt = routes(n, experts, topk)
    check(cuda, layer, w, xq, xs, idx, wt)
    layer.close()


def test_one_expert_has_them_all(cuda):
    layer, w = layer_of(cuda, 256, 128, 9, 1, limit=7)
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    xq, xs = ref.activations(500, 256, g)
    idx = torch.full((500, 1), 4, dtype=torch.int32, device="cuda")
    check(cuda, layer, w, xq, xs, idx, torch.ones(500, 1, device="cuda"))
    layer.close()


def test_routes_that_are_none_and_twice_the_same(cuda):
    layer, w = layer_of(cuda, 256, 256, 6, 3)
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    xq, xs = ref.activations(40, 256, g)
    idx, wt = routes(40, 6, 3)
    idx[::3, 0], idx[1, :], idx[2, 2] = -1, 6, 2 ** 31 - 1
    idx[4] = 5                               # the same expert three times
    out = check(cuda, layer, w, xq, xs, idx, wt)
    assert bool((out[1] == 0).all())         # no expert at all
    layer.close()


def test_an_expert_parallel_layer_adds_its_own(cuda):
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    xq, xs = ref.activations(60, 256, g)
    idx, wt = routes(60, 10, 4)
    for part in ((0, 4), (4, 10)):
        layer, w = layer_of(cuda, 256, 128, 10, 4, part=part)
        check(cuda, layer, w, xq, xs, idx, wt, lo=part[0])
        layer.close()


def test_broken_rows_stay_alone(cuda):
    layer, w = layer_of(cuda, 256, 128, 4, 2)
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    xq, xs = ref.activations(30, 256, g)
    idx, wt = routes(30, 4, 2)
    whole = torch.empty(30, 256, dtype=torch.bfloat16, device="cuda")
    layer.experts(xq, xs, idx, wt, whole)
    xq[5, 9], xs[11, 0] = 0xFF, 255
    out = torch.empty_like(whole)
    layer.experts(xq, xs, idx, wt, out)
    bad = torch.zeros(30, dtype=torch.bool, device="cuda")
    bad[5] = bad[11] = True
    assert bool(torch.isnan(out[bad]).all())
    assert torch.equal(out[~bad], whole[~bad])
    layer.close()


def test_captured(cuda):
    layer, w = layer_of(cuda, 256, 128, 12, 3)
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    xq, xs = ref.activations(90, 256, g)
    idx, wt = routes(90, 12, 3)
    out = torch.empty(90, 256, dtype=torch.bfloat16, device="cuda")
    work = torch.empty(layer.experts_workspace_bytes(90), dtype=torch.uint8, device="cuda")
    layer.experts(xq, xs, idx, wt, out, workspace=work)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.experts(xq, xs, idx, wt, out, workspace=work)
    for seed in (7, 8):
        idx.copy_(routes(90, 12, 3, seed)[0])
        out.fill_(5)
        graph.replay()
        torch.cuda.synchronize()
        y, b = want(w, xq, xs, idx, wt)
        assert bool(((out.double() - y).abs() <= b).all())
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(cuda.Dsv4CudaError, match="workspace"):
            layer.experts(xq, xs, idx, wt, out)
        out.fill_(1)
    layer.close()


def test_against_the_layers_forward(cuda):
    """The same routes through moe_forward (no shared expert): its BF16 boundaries (gate, up, h and
    a slot rounded to BF16, 2^-8 each at most) move the result by a few of those steps."""
    from oracle import make_moe_layer
    L = make_moe_layer(256, 128, 16, 2, seed=0)
    L["shared"] = None
    layer = cuda.MoeLayer(L, max_tokens=8)
    x = torch.randn(8, 256, generator=torch.Generator().manual_seed(0)).bfloat16().float().cuda()
    y = torch.empty_like(x)
    layer.forward(x, y)
    idx, wt, _ = layer.last_routes(8)
    q, s = ref.quantised(x.double())
    xq = (q.unflatten(1, (-1, 128)) / s[..., None]).flatten(1).to(torch.float8_e4m3fn).view(torch.uint8)
    xs = (torch.log2(s) + 127).to(torch.uint8)
    out = torch.empty(8, 256, dtype=torch.bfloat16, device="cuda")
    layer.experts(xq, xs, torch.tensor(idx).int().cuda(), torch.tensor(wt).float().cuda(), out)
    assert float((out.double() - y.double()).norm()) <= 0.03 * float(y.double().norm())
    layer.close()


def test_route_weights(cuda):
    """Zero, negative, tiny and huge ones; an infinity or NaN stays with its token."""
    layer, w = layer_of(cuda, 256, 256, 5, 2)
    g = torch.Generator(device="cuda")
    g.manual_seed(6)
    xq, xs = ref.activations(120, 256, g)
    idx, wt = routes(120, 5, 2)
    xq[3] = 0                                 # gate and up of zero, with a huge weight
    wt[::7, 0], wt[1::7], wt[2::7, 1] = 0.0, -2.5, 1e-30
    wt[3], wt[10, 0], wt[17] = 3e38, 1e-45, 1e12
    out = check(cuda, layer, w, xq, xs, idx, wt)
    assert bool((out[3] == 0).all())
    wt[40, 1], wt[41, 0] = float("inf"), float("nan")
    again = torch.empty_like(out)
    layer.experts(xq, xs, idx, wt, again)
    bad = torch.zeros(120, dtype=torch.bool, device="cuda")
    bad[40:42] = True
    assert bool(torch.isnan(again[bad]).all()) and torch.equal(again[~bad], out[~bad])
    layer.close()


@pytest.mark.parametrize("n,experts,topk,part", [(32, 300, 2, None), (33, 300, 2, None), (8, 1024, 8, None),
                                                 (11, 900, 6, (200, 870)), (400, 1000, 3, (1, 999))])
def test_many_experts(cuda, n, experts, topk, part):
    layer, w = layer_of(cuda, 128, 128, experts, topk, part=part)
    g = torch.Generator(device="cuda")
    g.manual_seed(7)
    xq, xs = ref.activations(n, 128, g)
    idx, wt = routes(n, experts, topk)
    check(cuda, layer, w, xq, xs, idx, wt, lo=part[0] if part else 0)
    layer.close()
