"""What the binding and the C entries refuse before anything is launched, without a GPU: routed
experts, grouped products, norm, latents' write, beams. Tensors are stand-ins that say they are on
one."""
import ctypes as C

import pytest
import torch

from test_paged_host import Fake

dsv4cuda = pytest.importorskip("dsv4cuda")
U8, I32, F32, BF = torch.uint8, torch.int32, torch.float32, torch.bfloat16


class On(Fake):
    """Fake, and the device that it is on."""

    def __init__(self, shape, dtype, stride=None, device=0):
        super().__init__(shape, dtype, stride)
        self.index = device

    def get_device(self):
        return self.index


@pytest.fixture
def calls(monkeypatch):
    """Library calls are written down, not made."""
    made = []
    for name in ("dsv4cuda_moe_experts", "dsv4cuda_grouped_gemm", "dsv4cuda_norm_quant",
                 "dsv4cuda_paged_write", "dsv4cuda_beam_select"):
        def call(*args, name=name):
            made.append((name, args))
            return 0
        monkeypatch.setattr(dsv4cuda.lib, name, call)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    return made


def norm(calls, **kw):
    a = dict(x=On((4, 256), BF), gain=On((256,), BF), codes=On((4, 256), U8), scales=On((4, 2), U8),
             residual=On((4, 256), BF, (300, 1)), sum_out=On((4, 256), BF), out=On((4, 256), BF), stream=0)
    a.update(kw)
    dsv4cuda.norm_quant(**a)


def test_norm(calls):
    norm(calls)
    shape = calls[0][1][7]._obj
    assert (shape.n_rows, shape.width, shape.bf16) == (4, 256, 1)
    assert (shape.x_stride, shape.residual_stride) == (256, 300)
    for bad in (dict(x=On((4, 256), torch.float16)), dict(x=On((4, 256), F32)),
                dict(x=On((4, 256), BF, (1, 4))), dict(x=On((4, 256), BF, (0, 1))),
                dict(x=On((256,), BF)), dict(x=On((4, 256), BF, device=1)),
                dict(residual=On((3, 256), BF)), dict(residual=On((4, 256), F32)),
                dict(sum_out=On((4, 256), BF, (100, 1))), dict(out=On((4, 255), BF)),
                dict(codes=On((4, 256), U8, device=1)), dict(out=On((4, 256), BF, device=1)),
                dict(gain=On((255,), BF)), dict(gain=On((256,), F32)), dict(codes=On((4, 255), U8)),
                dict(scales=On((4, 1), U8)), dict(codes=On((4, 256), torch.int8))):
        with pytest.raises(ValueError):
            norm(calls, **bad)
    assert len(calls) == 1
    norm(calls, x=On((1, 256), BF, (7, 1)), residual=None, sum_out=None, out=None)  # one row has no stride
    assert calls[1][1][7]._obj.x_stride == 0


def grouped(calls, **kw):
    a = dict(out=On((9, 100), BF), xq=On((5, 256), U8), xs=On((5, 2), U8), w=On((3, 100, 128), U8),
             ws=On((3, 100, 8), U8), offsets=On((4,), I32), src=On((9,), I32), dst=On((9,), I32), stream=0)
    a.update(kw)
    dsv4cuda.grouped_gemm(**a)


def test_grouped(calls):
    grouped(calls)
    grouped(calls, w=On((3, 100, 256), U8), ws=On((3, 1, 2), U8), src=None, out=On((9, 100), F32, (128, 1)))
    s = [c[1][8]._obj for c in calls]
    assert [(x.n_groups, x.n_rows, x.x_rows, x.out_rows, x.outs, x.width, x.fp8, x.bf16) for x in s] == [
        (3, 9, 5, 9, 100, 256, 0, 1), (3, 9, 5, 9, 100, 256, 1, 0)]
    assert s[1].out_stride == 128
    for bad in (dict(w=On((3, 100, 100), U8)), dict(w=On((3, 99, 128), U8)), dict(w=On((100, 128), U8)),
                dict(ws=On((3, 100, 7), U8)), dict(xs=On((5, 1), U8)), dict(offsets=On((3,), I32)),
                dict(dst=On((8,), I32)), dict(src=On((9,), torch.int64)),
                dict(out=On((9, 100), torch.float16)),
                dict(out=On((9, 100), BF, (50, 1))), dict(out=On((9, 100), BF, device=1)),
                dict(w=On((3, 100, 128), U8, device=1)), dict(workspace=On((1 << 20,), F32))):
        with pytest.raises(ValueError):
            grouped(calls, **bad)
    assert len(calls) == 2


def test_experts(calls):
    layer = object.__new__(dsv4cuda.MoeLayer)
    layer.hidden, layer.topk, layer.handle = 256, 2, None
    a = dict(xq=On((7, 256), U8), xs=On((7, 2), U8), idx=On((7, 2), I32), wt=On((7, 2), F32),
             out=On((7, 256), BF), stream=0)
    layer.experts(**a)
    assert calls[0][1][5] == 7
    for bad in (dict(xq=On((7, 128), U8)), dict(xq=On((7, 256), torch.int8)), dict(xs=On((7, 1), U8)),
                dict(idx=On((7, 2), torch.int64)), dict(wt=On((7, 1), F32)), dict(out=On((7, 256), F32)),
                dict(out=On((6, 256), BF)), dict(idx=On((7, 2), I32, device=1)),
                dict(xq=On((7, 256), U8, device=1))):
        with pytest.raises(ValueError):
            layer.experts(**{**a, **bad})
    layer.handle = C.c_void_p()


def test_write(calls):
    pool = object.__new__(dsv4cuda.PagedCache)
    pool.caches, pool._dims, pool._i64, pool._ref = [None, None], (448, 64), torch.int64, None
    pool.status_word = On((1,), I32)
    a = dict(layer=1, kv=On((5, 512), BF, (520, 1)), rows=On((5,), torch.int64), gain=On((512,), BF),
             rope_cos=On((5, 32), F32), rope_sin=On((5, 32), F32), stream=0)
    pool.write(**a)
    assert calls[0][1][1] == 1 and calls[0][1][4] == 520
    for bad in (dict(layer=2), dict(layer=-1), dict(kv=On((5, 448), BF)), dict(kv=On((5, 512), BF, (0, 1))),
                dict(rows=On((4,), torch.int64)), dict(rows=On((5,), I32)), dict(gain=On((448,), BF)),
                dict(rows=On((5,), torch.int64, device=1)), dict(rope_cos=On((4, 32), F32)),
                dict(rope_sin=On((5, 32), BF))):
        with pytest.raises(ValueError):
            pool.write(**{**a, **bad})


def beam(**kw):
    a = dict(logits=On((6, 50), BF, (64, 1)), score=On((2, 3), F32), parent=On((2, 4), I32),
             token=On((2, 4), I32), total=On((2, 4), F32), next=On((2, 3), I32), slot=On((2, 3), I32),
             dst=On((2, 3), I32), src=On((2, 3), I32), eos=7, stream=0)
    a.update(kw)
    dsv4cuda.beam_select(**a)


def test_beam(calls):
    beam()
    s = calls[0][1][9]._obj
    assert (s.n_groups, s.beams, s.n_cands, s.vocab, s.bf16, s.eos, s.stride) == (2, 3, 4, 50, 1, 7, 64)
    for bad in (dict(logits=On((5, 50), BF)), dict(logits=On((6, 50), BF, (0, 1))),
                dict(score=On((6,), F32)),
                dict(score=On((2, 3), BF)), dict(token=On((2, 3), I32)), dict(next=On((2, 2), I32)),
                dict(slot=On((2, 3), I32, device=1)), dict(total=On((2, 4), BF)),
                dict(dst=On((2, 2), I32)), dict(parent=On((8,), I32))):
        with pytest.raises(ValueError):
            beam(**bad)


# ------------------------------------------------------------ the C entries --

P = 1 << 20  # an address that is not read


def refused(rc, word):
    assert rc == -1 and word in dsv4cuda.last_error(), dsv4cuda.last_error()


def test_c_grouped():
    S, f = dsv4cuda.GroupedShape, dsv4cuda.lib.dsv4cuda_grouped_gemm
    good = (2, 10, 10, 10, 64, 256, 0, 1, 0)
    for i, v in ((0, 0), (0, 1025), (1, -1), (2, -1), (3, -1), (4, 0), (5, 0), (5, 200), (5,
    (1 << 20) + 128),
                 (8, 63)):
        bad = list(good)
        bad[i] = v
        refused(f(P, P, P, P, P, P, None, None, C.byref(S(*bad)), None, 0, None), "bad shape")
        assert dsv4cuda.lib.dsv4cuda_grouped_workspace_bytes(C.byref(S(*bad))) == 0
    refused(f(P, P, P, P, P, P, None, None, C.byref(S(1024, 10, 10, 10, 1 << 27, 256, 0, 1, 0)), None, 0,
    None),
            "bad shape")
    refused(f(P, P, P, P, P, P, None, None, C.byref(S(1, 1 << 21, 10, 10, 1 << 20, 256, 0, 1, 0)), None, 0,
    None),
            "bad shape")
    s = C.byref(S(*good))
    for args in ((None, P, P, P, P, P), (P, None, P, P, P, P), (P, P, P, P, P, None), (P, P + 8, P, P, P,
    P),
                 (P, P, P, P + 16, P, P), (P, P, P, P, P + 2, P), (P + 1, P, P, P, P, P)):
        refused(f(*args, None, None, s, None, 0, None), "bad arguments")
    assert f(None, None, None, None, None, None, None, None, C.byref(S(2, 0, 0, 0, 64, 256, 0, 1, 0)),
    None, 0,
             None) == 0  # nothing to do


def test_c_norm_and_beams():
    S, f = dsv4cuda.NormShape, dsv4cuda.lib.dsv4cuda_norm_quant
    for s in ((1, 0, 1, 1e-6), (1, 32769, 1, 1e-6), (-1, 8, 1, 1e-6), (1, 8, 1, 0.0), (1, 8, 1,
    float("nan")),
              (1, 8, 1, float("inf"))):
        refused(f(P, None, None, None, None, P, P, C.byref(S(*s)), None), "bad shape")
    ok = S(2, 8, 1, 1e-6)
    for args in ((None, None, None, None, None, P, P), (P, None, None, None, None, None, P),
                 (P, None, None, None, None, P, None), (P + 1, None, None, None, None, P, P),
                 (P, None, P + 1, None, None, P, P)):
        refused(f(*args, C.byref(ok), None), "bad arguments")
    refused(f(P, P, None, None, None, P, P, C.byref(S(2, 8, 1, 1e-6, 8, 7)), None), "bad arguments")
    assert f(None, None, None, None, None, None, None, C.byref(S(0, 8, 1, 1e-6)), None) == 0
    B, g = dsv4cuda.BeamShape, dsv4cuda.lib.dsv4cuda_beam_select
    for s in ((1, 0, 1, 9), (1, 33, 1, 9), (1, 1, 0, 9), (1, 1, 33, 9), (1, 1, 1, 0), (-1, 1, 1, 9),
              (1, 1, 1, 1 << 30), (1, 1, 1, 9, 1, -1, 8)):
        refused(g(P, P, P, P, P, P, None, None, None, C.byref(B(*s)), None), "bad shape")
    ok = B(1, 2, 2, 9, 1, -1, 0)
    refused(g(None, P, P, P, P, P, None, None, None, C.byref(ok), None), "bad arguments")
    refused(g(P + 1, P, P, P, P, P, None, None, None, C.byref(ok), None), "bad arguments")
    refused(g(P, P, P, P, P, P, P, None, None, C.byref(ok), None), "bad arguments")


def test_c_experts_of_no_layer():
    f = dsv4cuda.lib.dsv4cuda_moe_experts
    refused(f(None, P, P, P, P, 1, P, None, 0, None), "bad arguments")
    assert dsv4cuda.lib.dsv4cuda_moe_experts_workspace_bytes(None, 1) == 0
