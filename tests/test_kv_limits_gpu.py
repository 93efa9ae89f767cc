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
