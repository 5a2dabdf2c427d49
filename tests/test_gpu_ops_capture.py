"""Caches and rope tables that are collected while a graph is captured."""
import gc

import pytest
import torch

from test_gpu_kv4 import cache, ints, rows

pytestmark = pytest.mark.gpu


def test_a_capture_outlives_a_garbage_collection(gpu):
    from zerollm_amd._lib import ZLError
    from zerollm_amd.ops import KVCacheQ4, Rope
    c = cache(1, 2, 64, 500)
    k, q = rows(1, (1, 300, 2, 64)), rows(2, (1, 3, 4, 64))
    c.append(k, k, ints(0))
    pos, out = ints(200), torch.empty_like(q)
    work = torch.empty(c.work_bytes(1, 3, 4), dtype=torch.uint8, device="cuda")
    old = [KVCacheQ4(1, 2, 64, 500), Rope(64)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        old.clear()
        gc.collect()
        for bad in (lambda: Rope(64), c.close):
            with pytest.raises(ZLError, match="being captured"):
                bad()
        c.attend(q, pos, out=out, work=work)
    assert len(KVCacheQ4._gone) == 2
    for p in (200, 7, 290):
        pos.copy_(ints(p))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert (out == c.attend(q, ints(p))).all()
    Rope(64).close()
    assert not KVCacheQ4._gone
    c.close()
