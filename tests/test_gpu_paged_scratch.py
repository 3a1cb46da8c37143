"""The workspace that dsv4cuda_paged_attn keeps for calls that bring none: per thread and
stream, and gone with its thread."""
import threading
import time

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_thread_that_ends_leaves_no_workspace(cuda):
    """One token; the bounds ask for 64 slots of 16,384 positions, about 1 GB."""
    cache = cuda.LatentCache(64)
    pool = cuda.PagedCache.empty([cache], 64, 64, 256)
    pool.append(torch.zeros(1, dtype=torch.int32, device="cuda"),
                torch.ones(1, dtype=torch.int32, device="cuda"))
    q = torch.zeros(64, 64, 512, dtype=torch.bfloat16, device="cuda")
    out = torch.empty_like(q)
    q_start = torch.ones(65, dtype=torch.int32, device="cuda")
    q_start[0] = 0
    need = cuda.paged_attn_workspace_bytes(q, pool, 1, 16384)
    assert need > 1 << 30

    def call():
        cuda.paged_attn(out, q, pool, 0, q_start, 1, 16384, 1.0)
        torch.cuda.synchronize()
        held.append(torch.cuda.mem_get_info()[0])

    held = []
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    for _ in range(2):
        t = threading.Thread(target=call)
        t.start()
        t.join()
    assert before - held[0] >= need
    for _ in range(100):                # the system's thread ends a little after Python's
        if before - torch.cuda.mem_get_info()[0] < need // 2:
            break
        time.sleep(0.05)
    assert before - torch.cuda.mem_get_info()[0] < need // 2
