"""What the binding checks and passes on before a call of the paged cache, without a GPU:
tensors are stand-ins that say they are on one."""
import types

import pytest
import torch

dsv4cuda = pytest.importorskip("dsv4cuda")


class Fake:
    """The side of a CUDA tensor that the binding looks at."""

    def __init__(self, shape, dtype, stride=None, address=1 << 20):
        self.shape, self.dtype, self.address = tuple(shape), dtype, address
        self.strides = stride
        if stride is None:
            self.strides, n = (), 1
            for k in reversed(self.shape):
                self.strides, n = (n, *self.strides), n * k
        self.is_cuda, self.device = True, "cuda"

    def stride(self, i=None):
        return self.strides if i is None else self.strides[i]

    def dim(self):
        return len(self.shape)

    def numel(self):
        n = 1
        for k in self.shape:
            n *= k
        return n

    def element_size(self):
        return self.dtype.itemsize

    def is_contiguous(self):
        return self.strides == Fake(self.shape, self.dtype).strides

    def data_ptr(self):
        return self.address if self.numel() else 0


@pytest.fixture
def calls(monkeypatch):
    """Library calls are written down, not made."""
    made = []

    def record(name):
        def call(*args):
            made.append((name, args))
            return 0
        return call
    for name in ("dsv4cuda_paged_fork", "dsv4cuda_paged_append", "dsv4cuda_paged_attn"):
        monkeypatch.setattr(dsv4cuda.lib, name, record(name))
    return made


@pytest.fixture
def pool():
    p = dsv4cuda.PagedCache.__new__(dsv4cuda.PagedCache)
    p._i32, p._i64 = torch.int32, torch.int64
    p._ref, p.n_seqs = types.SimpleNamespace(), 4
    return p


def test_free_reads_nothing_that_another_stream_writes(calls, pool):
    """No array of sources is made: it would be filled on torch's current stream, and
    the call is made on the given one."""
    slots = Fake([3], torch.int32)
    pool.free(slots, stream=77)
    assert calls == [("dsv4cuda_paged_fork", (pool._ref, slots.address, None, 3, 77))]


def attn(pool, q, out, **kw):
    dsv4cuda.paged_attn(out, q, pool, 0, Fake([pool.n_seqs + 1], torch.int32), 4, 64, 1.0,
                        stream=77, **kw)


@pytest.mark.parametrize("stride", [0, 4 * 512 - 8])
@pytest.mark.parametrize("which", ["q", "out"])
def test_rows_that_overlap_are_refused(calls, pool, which, stride):
    """One row expanded to several, or rows that begin inside the one before."""
    whole, over = Fake([3, 4, 512], torch.bfloat16), \
        Fake([3, 4, 512], torch.bfloat16, (stride, 512, 1))
    with pytest.raises(ValueError, match="overlap"):
        attn(pool, *((over, whole) if which == "q" else (whole, over)))
    if which == "q":
        with pytest.raises(ValueError, match="overlap"):
            dsv4cuda.paged_attn_workspace_bytes(over, pool, 4, 64)
    assert not calls


def test_the_stride_of_a_single_row_does_not_matter(calls, pool):
    one = Fake([1, 4, 512], torch.bfloat16, (0, 512, 1))
    attn(pool, one, Fake([1, 4, 512], torch.bfloat16))
    apart = Fake([3, 4, 512], torch.bfloat16, (4 * 512 + 8, 512, 1))
    attn(pool, apart, Fake([3, 4, 512], torch.bfloat16))
    assert len(calls) == 2


@pytest.mark.parametrize("workspace", [
    torch.empty(1 << 20, dtype=torch.uint8),                        # not on the GPU
    Fake([1 << 20], torch.float32), Fake([1 << 20], torch.int8),
    Fake([1 << 20], torch.uint8, (2,))], ids=["host", "fp32", "int8", "every other byte"])
def test_a_workspace_that_is_none(calls, pool, workspace):
    q = Fake([3, 4, 512], torch.bfloat16)
    with pytest.raises(ValueError, match="workspace"):
        attn(pool, q, q, workspace=workspace)
    assert not calls
    good = Fake([1 << 20], torch.uint8, address=1 << 30)
    attn(pool, q, q, workspace=good)
    assert calls[0][1][-3:] == (1 << 30, 1 << 20, 77)
