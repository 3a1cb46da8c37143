"""MoeLayer.experts holds its tensors to the layer's own device. Without a GPU: tensors are stand-ins
that say they are on one."""
import pytest
import torch

from test_operators_host import BF, F32, I32, On, U8, calls, dsv4cuda  # noqa: F401


def call(layer):
    layer.experts(xq=On((7, 256), U8), xs=On((7, 2), U8), idx=On((7, 2), I32), wt=On((7, 2), F32),
                  out=On((7, 256), BF), stream=0)


def test_a_layer_of_another_device(calls):  # noqa: F811
    layer = object.__new__(dsv4cuda.MoeLayer)
    layer.hidden, layer.topk, layer.handle = 256, 2, None
    layer.on = 1
    with pytest.raises(ValueError, match="cuda:1"):
        call(layer)
    assert not calls
    layer.on = 0
    call(layer)
    assert len(calls) == 1


def test_the_layer_knows_where_its_weights_are(monkeypatch):
    monkeypatch.setattr(dsv4cuda.lib, "dsv4cuda_moe_create_device", lambda *a: 0)
    monkeypatch.setattr(dsv4cuda.lib, "dsv4cuda_moe_destroy", lambda *a: None)
    names = ("gate_w", "w1", "s1", "w3", "s3", "w2", "s2")

    class Weights(On):
        def data_ptr(self):
            return 1 << 20
    weights = {n: Weights((4, 4), torch.uint8, device=1) for n in names}
    layer = dsv4cuda.MoeLayer(dict(hidden=256, moe_inter=128, n_experts=4, topk=2, swiglu_limit=10,
                                   route_scale=1.0, **weights), device=True)
    assert layer.on == 1
