"""What dsv4cuda_moe_experts refuses of a layer, before anything is launched."""
import pytest
import torch

import grouped_ref as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("missing", ["w1", "s1", "w3", "s3", "w2", "s2"])
def test_a_layer_without_one_of_its_experts_weights(cuda, missing):
    """Adopted weights may be absent (a layer that only routes): nothing is read there."""
    g = torch.Generator(device="cuda")
    g.manual_seed(0)
    e, h, i, k, n = 4, 256, 128, 2, 3
    weights = dict(gate_w=torch.zeros(e, h, dtype=torch.int16, device="cuda"))
    weights["w1"], weights["s1"] = ref.fp4(e, i, h, g)
    weights["w3"], weights["s3"] = ref.fp4(e, i, h, g)
    weights["w2"], weights["s2"] = ref.fp4(e, h, i, g)
    xq, xs = ref.activations(n, h, g)
    idx = torch.tensor([[0, 1], [1, 3], [2, 3]], dtype=torch.int32, device="cuda")
    wt = torch.full((n, k), 0.5, device="cuda")
    sizes = dict(hidden=h, moe_inter=i, n_experts=e, topk=k, swiglu_limit=10, route_scale=1.0)
    out = torch.full((n, h), 7.0, dtype=torch.bfloat16, device="cuda")
    layer = cuda.MoeLayer(dict(sizes, **{**weights, missing: None}), max_tokens=1, device=True)
    with pytest.raises(RuntimeError, match="no routed experts"):
        layer.experts(xq, xs, idx, wt, out)
    assert bool((out == 7).all())
    layer.close()
    layer = cuda.MoeLayer(dict(sizes, **weights), max_tokens=1, device=True)
    layer.experts(xq, xs, idx, wt, out)
    assert bool(torch.isfinite(out).all()) and not bool((out == 7).all())
    layer.close()
