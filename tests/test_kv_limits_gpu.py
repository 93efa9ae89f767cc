"""Calls at the edges of what the cache's entries take: many sequences, adjacent buffers, workspaces
that grow."""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu

D = 128


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def test_export_of_many_sequences():
    """More sequences than a grid has rows."""
    from ferrisres_b200 import paged
    g = generator(1)
    c = paged.PagedKv3Cache(1, 8, 2)
    rids = [c.create_request() for _ in range(2)]
    c.append(0, rids, *[torch.randn((2, 70, 2, D), generator=g, device="cuda") for _ in range(2)])
    want = c.export_range(0, rids, 30, 34)
    got = c.export_range(0, rids * 40000, 30, 34)
    for a, b in zip(want, got):
        assert b.shape[0] == 80000 and torch.equal(b.view(40000, 2, *a.shape[1:]), a.expand(40000, *a.shape))
    c.ctx.check()
    c.close()


def test_select_beside_other_memory():
    """Weight rows that are a part of wider ones end before the last row's pitch does: what lies there
    may be the output."""
    from ferrisres_b200 import kv
    from ferrisres_b200._lib import ShapeError, call
    from ferrisres_b200.gpu import _stream_ptr, get_context
    g = generator(2)
    n, pitch, keep = 63, 128, 20
    buf = torch.zeros(1024, device="cuda")
    w = buf[37:37 + 2 * pitch].view(1, 2, pitch)[:, :, :n]
    w.copy_(torch.rand((1, 2, n), generator=g, device="cuda"))
    idx = torch.empty((1, 2, keep), dtype=torch.int32, device="cuda")
    want_idx, want = kv.select_heavy(w.clone(), keep, 4)

    def go(at):
        call("ft_kv_select_heavy", get_context().handle, 1, 2, C.c_void_p(w.data_ptr()), pitch, None, n, keep, 4,
             C.c_void_p(idx.data_ptr()), C.c_void_p(buf.data_ptr() + 4 * at), keep, _stream_ptr())

    behind = 37 + pitch + n  # the first entry behind the last row
    go(behind)
    assert torch.equal(idx, want_idx)
    assert torch.equal(buf[behind:behind + 2 * keep].view(1, 2, keep), want[:, :, :keep])
    for at in (behind - 1, 37 - 2 * keep + 1):
        with pytest.raises(ShapeError):
            go(at)
