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


def free_bytes():
    torch.cuda.synchronize()
    return torch.cuda.mem_get_info()[0]


def test_a_workspace_that_grows_takes_what_it_needs():
    """The scores of a decode with weights over 64 more positions: an eighth more memory at most, not a
    second buffer of twice the size beside the first."""
    from ferrisres_b200 import kv
    n, Hq = 8192, 4096
    c = kv.Kv3Cache(1, 1, n + 128)
    x = torch.zeros((1, n, 1, D), device="cuda")
    c.append(x, x)
    q = torch.zeros((1, Hq, D), device="cuda")
    out, w = torch.empty_like(q), torch.zeros((1, 1, n + 64), device="cuda")
    c.flash_decode(q, weights=w, out=out)
    scores = 4 * Hq * n
    c.append(x[:, :64], x[:, :64])
    before = free_bytes()
    c.flash_decode(q, weights=w, out=out)
    assert before - free_bytes() <= 0.25 * scores
    c.close()


def test_a_captured_workspace_stays():
    """A graph keeps the buffers that it was captured with, however often calls outside it need larger
    ones."""
    from ferrisres_b200 import kv
    g = generator(3)
    c = kv.Kv3Cache(1, 2, 4096)
    x = [torch.randn((1, 4000, 2, D), generator=g, device="cuda") for _ in range(2)]
    c.append(x[0][:, :300], x[1][:, :300])
    q = torch.randn((1, 8, D), generator=g, device="cuda")
    t = torch.randn((1, 5, 8, D), generator=g, device="cuda")
    w = torch.zeros((1, 2, 4096), device="cuda")
    want = [c.flash_decode(q, weights=w), c.tree_decode(t)]
    out = [torch.empty_like(a) for a in want]

    def calls():
        c.flash_decode(q, weights=w, out=out[0])
        c.tree_decode(t, out=out[1])

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls()
    for n in (400, 900, 2100):
        c.append(*[y[:, :n] for y in x])
        calls()
        big = torch.zeros((1, 64, 8, D), device="cuda")
        c.tree_decode(big)
        # what the cache gave back would be overwritten here
        junk = [torch.full((1 << 20,), float("nan"), device="cuda") for _ in range(8)]
        for o in out:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        del junk
    c.ctx.check()
    c.close()
