"""PagedCache.free on a stream of its own."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_free_on_another_stream_than_the_current_one(cuda):
    """The current stream is busy meanwhile; nothing of the call waits for it."""
    pool = cuda.PagedCache.empty([cuda.LatentCache(64, 64, 2)], 4, 6, 4)
    i32 = dict(dtype=torch.int32, device="cuda")
    pool.append(torch.arange(6, **i32), torch.tensor([5, 1, 9, 4, 16, 2], **i32))
    slots = torch.tensor([4, 0, 2], **i32)
    side = torch.cuda.Stream()
    busy = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    for _ in range(20):
        busy = (busy @ busy).clamp_(-1, 1)
    pool.free(slots, stream=side.cuda_stream)
    side.synchronize()
    torch.cuda.synchronize()
    assert pool.length.tolist() == [0, 1, 0, 4, 0, 2]
    assert pool.table.tolist() == [[-1] * 4, [2, -1, -1, -1], [-1] * 4, [6, -1, -1, -1],
                                   [-1] * 4, [11, -1, -1, -1]]
    want = [0] * 16
    for q in (2, 6, 11):
        want[q] = 1
    assert pool.refs.tolist() == want and pool.status() == 0


def test_free_refuses_what_fork_refuses(cuda):
    pool = cuda.PagedCache.empty([cuda.LatentCache(64, 64, 2)], 4, 3, 4)
    i32 = dict(dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        pool.free(torch.zeros(1, dtype=torch.int64, device="cuda"))
    with pytest.raises(cuda.Dsv4CudaError, match="one op per slot"):
        pool.free(torch.zeros(4, **i32))
    pool.append(torch.tensor([0, 1], **i32), torch.tensor([3, 4], **i32))
    pool.free(torch.tensor([1, 1, 9], **i32))       # named twice, out of range
    assert pool.length.tolist() == [3, 0, 0] and pool.status() == pool.BAD_OP
    pool.free(torch.zeros(0, **i32))
    assert pool.length.tolist() == [3, 0, 0] and pool.status() == 0
