"""A process whose first call of an operator is captured into a graph: what the library makes for
itself by then (the device's error word among it) does not end the capture, and the graph gives what
an eager call gives."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.join(os.path.dirname(HERE), "deepseek-v4-flash-0731-in-c_b200")

START = f"""
import sys
sys.path[:0] = [{HERE!r}, {PKG!r}]
import torch
import dsv4cuda as cuda
import grouped_ref as ref
g = torch.Generator(device="cuda")
g.manual_seed(0)
u8, i32 = dict(dtype=torch.uint8, device="cuda"), dict(dtype=torch.int32, device="cuda")

def captured(call, outs):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    graph.replay()
    torch.cuda.synchronize()
    got = [o.clone() for o in outs]
    for o in outs:
        o.zero_()
    call()
    torch.cuda.synchronize()
    for a, b in zip(got, outs):
        assert torch.equal(a, b)
    assert any(bool((a != 0).any()) for a in got)
    assert cuda.device_error() == 0
    print("equal")
"""

CALLS = dict(
    grouped="""
xq, xs = ref.activations(40, 256, g)
w, ws = ref.fp4(3, 200, 256, g)
offsets = torch.tensor([0, 11, 11, 40], **i32)
out = torch.empty(40, 200, device="cuda")
work = torch.empty(cuda.grouped_workspace_bytes(out, xq, w, 40), **u8)
captured(lambda: cuda.grouped_gemm(out, xq, xs, w, ws, offsets, workspace=work), [out])
""",
    experts="""
e, h, i, k, n = 8, 256, 128, 2, 90
weights = dict(gate_w=torch.zeros(e, h, dtype=torch.int16, device="cuda"))
weights["w1"], weights["s1"] = ref.fp4(e, i, h, g)
weights["w3"], weights["s3"] = ref.fp4(e, i, h, g)
weights["w2"], weights["s2"] = ref.fp4(e, h, i, g)
layer = cuda.MoeLayer(dict(hidden=h, moe_inter=i, n_experts=e, topk=k, swiglu_limit=10, route_scale=1.0,
                           **weights), max_tokens=1, device=True)
xq, xs = ref.activations(n, h, g)
idx = torch.randint(0, e, (n, k), **i32, generator=g)
wt = torch.rand(n, k, device="cuda", generator=g)
out = torch.empty(n, h, dtype=torch.bfloat16, device="cuda")
work = torch.empty(layer.experts_workspace_bytes(n), **u8)
captured(lambda: layer.experts(xq, xs, idx, wt, out, workspace=work), [out])
""",
    norm="""
x = torch.randn(9, 500, device="cuda", generator=g)
codes, scales = torch.empty(9, 500, **u8), torch.empty(9, 4, **u8)
captured(lambda: cuda.norm_quant(x, None, codes, scales), [codes, scales])
""",
    write="""
cache = cuda.LatentCache(64)
pool = cuda.PagedCache.empty([cache], 16, 2, 4)
kv = torch.randn(5, 512, device="cuda", generator=g)
rows = torch.tensor([3, 60, -1, 17, 0], device="cuda")
captured(lambda: pool.write(0, kv, rows), [cache.codes, cache.scales, cache.rope])
""",
    beam="""
x = torch.randn(6, 9000, device="cuda", generator=g)
score = -torch.rand(2, 3, device="cuda", generator=g)
parent, token, total = torch.empty(2, 4, **i32), torch.empty(2, 4, **i32), torch.empty(2, 4, device="cuda")
nxt = torch.empty(2, 3, **i32)
captured(lambda: cuda.beam_select(x, score, parent, token, total, nxt), [parent, token, total, nxt])
""")


@pytest.mark.parametrize("name", CALLS)
def test_first_call_captured(name):
    r = subprocess.run([sys.executable, "-c", START + CALLS[name]], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "equal" in r.stdout, r.stderr[-3000:]
