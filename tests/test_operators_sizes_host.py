"""Sizes that the C entries' ints do not hold are refused by the binding, not cut off: a call of 2^32 + 5
rows would else be one of 5. Without a GPU: tensors are stand-ins that say they are on one."""
import pytest
import torch

import test_operators_host as host
from test_operators_host import BF, F32, I32, On, U8, calls, dsv4cuda  # noqa: F401

LONG = (1 << 32) + 5  # 5, cut off
HALF = 1 << 31        # the first that is none


@pytest.mark.parametrize("n", [LONG, HALF])
def test_rows(calls, n):  # noqa: F811
    with pytest.raises(ValueError, match="31 bits"):
        host.norm(calls, x=On((n, 1), BF), gain=None, codes=On((n, 1), U8), scales=On((n, 1), U8),
                  residual=None, sum_out=None, out=None)
    layer = object.__new__(dsv4cuda.MoeLayer)
    layer.hidden, layer.topk, layer.handle = 128, 1, None
    with pytest.raises(ValueError, match="31 bits"):
        layer.experts(On((n, 128), U8), On((n, 1), U8), On((n, 1), I32), On((n, 1), F32), On((n, 128), BF),
                      stream=0)
    with pytest.raises(ValueError, match="31 bits"):
        layer.experts_workspace_bytes(n)
    pool = object.__new__(dsv4cuda.PagedCache)
    pool.caches, pool._dims, pool._i64, pool._ref = [None], (64, 0), torch.int64, None
    pool.status_word = On((1,), I32)
    with pytest.raises(ValueError, match="31 bits"):
        pool.write(0, On((n, 64), BF), On((n,), torch.int64), stream=0)
    assert not calls


@pytest.mark.parametrize("n", [LONG, HALF])
@pytest.mark.parametrize("which", ["outs", "x", "out", "src"])
def test_grouped(calls, n, which):  # noqa: F811
    outs = n if which == "outs" else 64
    rows = n if which in ("out", "src") else 4
    x = n if which == "x" else 4
    out = On((rows if which == "out" else 4, outs), BF)
    xq, w = On((x, 128), U8), On((1, outs, 64), U8)
    src = On((n,), I32) if which == "src" else On((4,), I32)
    with pytest.raises(ValueError, match="31 bits"):
        dsv4cuda.grouped_gemm(out, xq, On((x, 1), U8), w, On((1, outs, 4), U8), On((2,), I32), src=src,
                              stream=0)
    with pytest.raises(ValueError, match="31 bits"):
        dsv4cuda.grouped_workspace_bytes(out, xq, w, src.numel())
    assert not calls


@pytest.mark.parametrize("eos", [LONG, HALF, -HALF - 1])
def test_beams_end(calls, eos):  # noqa: F811
    with pytest.raises(ValueError, match="31 bits"):
        host.beam(eos=eos)
    with pytest.raises(ValueError, match="31 bits"):
        host.beam(logits=On((6, LONG), BF))
    assert not calls
    host.beam(eos=HALF - 1)
    assert calls[0][1][9]._obj.eos == HALF - 1
