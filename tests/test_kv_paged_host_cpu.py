"""Host side of the paged cache's calls, without a GPU: pages, reference counts and registered
prefixes around keep, append and eviction, and what a call on another stream waits for."""
import types

import pytest
import torch

from ferrisres_b200 import kv, paged
from ferrisres_b200._lib import OOMError, ShapeError, UnsupportedError
from ferrisres_b200.paged import PAGE_POSITIONS, PagedAttentionManager, PagedKv3Cache

NOT_CAPTURED = PagedKv3Cache._not_captured


@pytest.fixture
def host(monkeypatch):
    """make(num_pages): a cache on the CPU whose C calls are recorded, not made."""
    seen = types.SimpleNamespace(calls=[], used=[], ordered=[])

    def dptr(t):
        seen.used.append(t)
        return None

    def call_stream(device, stream, *tensors):
        seen.ordered.append((stream, [t for t in tensors if t is not None], len(seen.calls)))
        return None

    for m in (kv, paged):
        monkeypatch.setattr(m, "call", lambda name, *a: seen.calls.append((name, a)))
        monkeypatch.setattr(m, "_dptr", dptr)
        monkeypatch.setattr(m, "_call_stream", call_stream)
    monkeypatch.setattr(PagedKv3Cache, "_not_captured", staticmethod(lambda *a: None))

    def make(num_pages, kv_heads=2, num_layers=1):
        c = PagedKv3Cache.__new__(PagedKv3Cache)
        c.manager = PagedAttentionManager(num_layers, num_pages, PAGE_POSITIONS, kv_heads * 128)
        c.ctx = types.SimpleNamespace(handle=None)
        c.device, c.kv_heads, c.mode, c.handle = torch.device("cpu"), kv_heads, "R", None
        return c

    make.seen = seen
    return make


def fill(c, n, layer=0):
    r = c.create_request()
    x = torch.zeros((1, n, c.kv_heads, 128))
    c.append_packed(layer, [r], *packed(c, 1, n))
    assert c.seq_len(r, layer) == n and x.shape[1] == n
    return r


def packed(c, batch, n):
    codes = torch.zeros((batch, n, c.kv_heads * 48), dtype=torch.uint8)
    mm = torch.zeros((batch, n, c.kv_heads, 2))
    return codes, mm, codes.clone(), mm.clone()


def idx(n, start=0):
    return torch.arange(start, start + n, dtype=torch.int32)


def state(c, rids):
    """Everything that a refused call has to leave as it was."""
    a = c.manager.allocator
    return ([(c.block_table(r), c.seq_len(r)) for r in rids], list(a._ref), sorted(a._free))


# ------------------------------------------------------- registered prefixes --
def test_keep_forgets_a_prefix_whose_pages_it_rewrites(host):
    c = host(8)
    r = fill(c, 100)
    pm = c.manager.prefix_manager()
    tokens = list(range(64))
    pm.register_prefix(tokens, [c.block_table(r)[:2]])
    pm.register_prefix([7] * 32, [c.block_table(r)[:1]])
    # positions from 70 on: neither prefix has any
    c.keep(0, [r], idx(10, 80), starts=[70])
    assert pm.has_prefix(tokens) and pm.has_prefix([7] * 32)
    # from 40 on: the second page of the first
    c.keep(0, [r], idx(20, 50), starts=[40])
    assert pm.lookup_prefix(tokens) is None and pm.has_prefix([7] * 32)
    c.keep(0, [r], idx(30, 20), starts=[0])
    assert pm.lookup_prefix([7] * 32) is None


def test_keep_forgets_a_prefix_whose_pages_it_frees(host):
    c = host(8)
    r = fill(c, 128)
    pm = c.manager.prefix_manager()
    pm.register_prefix(range(128), [c.block_table(r)])
    pm.register_prefix(range(64), [c.block_table(r)[:2]])
    c.keep(0, [r], idx(0), starts=[64])  # nothing moves, two pages go
    assert pm.lookup_prefix(range(128)) is None and pm.has_prefix(range(64))
    assert c.manager.num_free_blocks() == 6


def test_a_partly_filled_page_keeps_its_prefix(host):
    """A prefix of 40 positions: positions from 40 on may change in its second page."""
    c = host(8)
    r = fill(c, 60)
    pm = c.manager.prefix_manager()
    pm.register_prefix(range(40), [c.block_table(r)])
    c.keep(0, [r], idx(5, 50), starts=[40])
    assert pm.has_prefix(range(40))
    c.keep(0, [r], idx(3, 41), starts=[39])
    assert not pm.has_prefix(range(40))


def test_a_prefix_beyond_the_new_end_is_forgotten(host):
    """Positions 50 and up go: the next append writes over them in the second page."""
    c = host(8)
    r = fill(c, 64)
    pm = c.manager.prefix_manager()
    pages = c.block_table(r)
    pm.register_prefix(range(64), [pages])
    pm.register_prefix(range(50), [pages])
    pm.register_prefix(range(32), [pages[:1]])
    c.keep(0, [r], idx(0), starts=[64])  # all stay
    assert pm.num_prefixes() == 3
    c.keep(0, [r], idx(0), starts=[50])
    assert pm.lookup_prefix(range(64)) is None and pm.has_prefix(range(50)) and pm.has_prefix(range(32))


def test_keep_spares_a_prefix_that_others_hold(host):
    c = host(8)
    r = fill(c, 64)
    pm = c.manager.prefix_manager()
    pages = c.block_table(r)
    pm.register_prefix(range(64), [pages])
    assert pm.lookup_prefix(range(64)) == [pages]  # another user of the pages
    c.keep(0, [r], idx(40, 10))
    assert [n for n, _ in host.seen.calls][-2:] == ["ft_kvp_copy_pages", "ft_kvp_keep"]
    assert not set(c.block_table(r)) & set(pages)
    assert pm.lookup_prefix(range(64)) == [pages]


def test_evict_forgets_a_prefix(host, monkeypatch):
    c = host(8)
    r = fill(c, 64)
    pm = c.manager.prefix_manager()
    pm.register_prefix(range(32), [c.block_table(r)[:1]])
    monkeypatch.setattr(paged, "select_heavy", lambda w, n, *a, **k: (idx(n).expand(1, 2, n), w))
    c.evict_heavy(0, [r], torch.zeros((1, 2, 64)), 64)  # nothing to evict
    assert pm.has_prefix(range(32))
    c.evict_heavy(0, [r], torch.zeros((1, 2, 64)), 40)
    assert pm.lookup_prefix(range(32)) is None


def test_forgetting_looks_at_the_pages_of_the_call_only(host):
    """Registrations anew, removed, of several layers and in large numbers."""
    c = host(8)
    r, other = fill(c, 64), fill(c, 64)
    pm = c.manager.prefix_manager()
    a, b = c.block_table(r), c.block_table(other)
    for i in range(500):
        pm.register_prefix([i] * 64, [b])
    pm.register_prefix(range(64), [a])
    pm.register_prefix(range(64), [b])  # the same tokens, now elsewhere
    pm.register_prefix(range(32), [b[:1], a[:1]])  # the second layer's page
    pm.register_prefix(range(33), [a])
    pm.remove_prefix(range(33))
    pm.remove_prefix(range(33))
    c.keep(0, [r], idx(10, 5))
    assert not pm.has_prefix(range(32)) and not pm.has_prefix(range(33))
    assert pm.has_prefix(range(64)) and pm.num_prefixes() == 501
    c.keep(0, [other], idx(10, 5))
    assert pm.num_prefixes() == 0 and not pm._named


# ------------------------------------------------------------- free pages --
def test_keep_needs_no_copy_for_the_last_owner(host):
    """A request and its fork, both rewritten: half of their pages have to be copied."""
    c = host(4)
    a = fill(c, 64)
    b = c.fork_request(a)
    assert c.manager.num_free_blocks() == 2
    c.keep(0, [a, b], idx(40, 10))
    assert not set(c.block_table(a)) & set(c.block_table(b))
    assert c.seq_len(a) == c.seq_len(b) == 40


def test_keep_refuses_before_it_changes_anything(host):
    c = host(4)
    a = fill(c, 64)
    b = c.fork_request(a)
    d = fill(c, 10)
    before = state(c, [a, b, d])
    with pytest.raises(OOMError):
        c.keep(0, [a, b], idx(40, 10))
    with pytest.raises(OOMError):  # the other owner is not part of the call
        c.keep(0, [b], idx(40, 10))
    assert state(c, [a, b, d]) == before
    c.keep(0, [b], idx(8, 3), counts=[8])  # one page to write, one free
    assert c.seq_len(b) == 8


# -------------------------------------------------------------------- append --
def values(c, batch, n):
    return torch.zeros((batch, n, c.kv_heads, 128)), torch.zeros((batch, n, c.kv_heads, 128))


@pytest.mark.parametrize("how", ["append", "append_packed"])
def test_append_refuses_before_it_changes_anything(host, how):
    c = host(4)
    a = fill(c, 40)
    b = c.fork_request(a)
    d = c.create_request()
    before, calls = state(c, [a, b, d]), len(host.seen.calls)
    data = {"append": values, "append_packed": packed}[how]
    with pytest.raises(OOMError):
        # b: a copy of the shared page; d: two pages; two are free
        getattr(c, how)(0, [b, d], *data(c, 2, 64))
    with pytest.raises(ShapeError):
        getattr(c, how)(0, [b, 99], *data(c, 2, 4))
    assert state(c, [a, b, d]) == before and len(host.seen.calls) == calls
    # a request and its fork: one of the two copies the page
    getattr(c, how)(0, [a, b], *data(c, 2, 24))
    assert c.seq_len(a) == c.seq_len(b) == 64
    assert c.block_table(a)[0] == c.block_table(b)[0] and c.block_table(a)[1] != c.block_table(b)[1]
    assert c.manager.num_free_blocks() == 1


# ------------------------------------------------------------- other streams --
def pool_calls(c):
    r = fill(c, 70)
    f = c.fork_request(r)
    q = torch.zeros((1, 4, 128))
    return {
        "append": lambda s: c.append(0, [f], *(t[:, ::2] for t in values(c, 1, 8)), stream=s),
        "append_packed": lambda s: c.append_packed(0, [f], *(t[:, ::2] for t in packed(c, 1, 8)), stream=s),
        "keep": lambda s: c.keep(0, [f], idx(9, 40), starts=[33], stream=s),
        "tree_decode": lambda s: c.tree_decode(0, [r], torch.zeros((1, 3, 4, 128)), stream=s),
        "flash_decode": lambda s: c.flash_decode(0, [r], q, stream=s),
        "weights": lambda s: c.flash_decode(0, [r], q, weights=torch.zeros((1, 2, 70)), stream=s),
        "get_range": lambda s: c.get_range(0, [r], 3, 50, stream=s),
        "export_range": lambda s: c.export_range(0, [r], 3, 50, stream=s),
    }


def ring(host):
    c = kv.Kv3Cache.__new__(kv.Kv3Cache)
    c.ctx = types.SimpleNamespace(handle=None)
    c.device, c.batch, c.kv_heads, c.handle = torch.device("cpu"), 2, 2, None
    return c


def ring_calls(c):
    x = torch.zeros((2, 8, 2, 128))
    codes = torch.zeros((2, 8, 96), dtype=torch.uint8)
    mm = torch.zeros((2, 8, 2, 2))
    q = torch.zeros((2, 4, 128))
    return {
        "append": lambda s: c.append(x[:, ::2], x[:, 1::2], stream=s),
        "append_packed": lambda s: c.append_packed(codes[:, ::2], mm[:, ::2], codes[:, 1::2], mm[:, 1::2], stream=s),
        "get_range": lambda s: c.get_range(3, 50, stream=s),
        "export_range": lambda s: c.export_range(3, 50, stream=s),
        "flash_decode": lambda s: c.flash_decode(q, stream=s),
        "tree_decode": lambda s: c.tree_decode(torch.zeros((2, 3, 4, 128)), stream=s),
        "keep": lambda s: c.keep(idx(9), stream=s),
    }


@pytest.mark.parametrize("name", ["append", "append_packed", "keep", "tree_decode", "flash_decode", "weights",
                                  "get_range", "export_range"])
def test_paged_calls_are_ordered_behind_the_current_stream(host, name):
    """Every tensor that a call hands over is ordered with, and held for, the stream that it runs on,
    before anything is launched there."""
    c = host(16)
    go = pool_calls(c)[name]
    host.seen.calls.clear(), host.seen.used.clear(), host.seen.ordered.clear()
    side = object()
    go(side)
    check_ordered(host.seen, side)


@pytest.mark.parametrize("name", ["append", "append_packed", "get_range", "export_range", "flash_decode", "tree_decode",
                                  "keep"])
def test_ring_calls_are_ordered_behind_the_current_stream(host, name):
    go = ring_calls(ring(host))[name]
    side = object()
    go(side)
    check_ordered(host.seen, side)


def check_ordered(seen, side):
    launches = [i for i, (n, _) in enumerate(seen.calls)]
    assert launches and len(seen.ordered) >= 1
    assert all(s is side for s, _, _ in seen.ordered)
    assert len(seen.ordered) == len(launches)  # one for every launch
    held = {t.untyped_storage().data_ptr() for _, ts, _ in seen.ordered for t in ts}
    for t in seen.used:
        assert t.numel() == 0 or t.untyped_storage().data_ptr() in held, tuple(t.shape)


# ----------------------------------------------------------- captured streams --
@pytest.mark.parametrize("current,given", [(True, None), (True, False), (False, True)])
@pytest.mark.parametrize("name", ["append", "append_packed", "keep", "tree_decode", "flash_decode", "weights",
                                  "get_range", "export_range", "evict_heavy"])
def test_calls_refuse_a_captured_stream(host, monkeypatch, name, current, given):
    """The current stream or the one given is being captured: refused before anything changes or runs."""
    c = host(16)
    go = {**pool_calls(c), "evict_heavy": lambda s: c.evict_heavy(0, [0], torch.zeros((1, 2, 70)), 40, stream=s)}[name]
    monkeypatch.setattr(PagedKv3Cache, "_not_captured", staticmethod(NOT_CAPTURED))
    now = [current]

    class On:
        def __init__(self, s):
            self.to, self.was = s, now[0]

        def __enter__(self):
            now[0] = self.to

        def __exit__(self, *a):
            now[0] = self.was

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "stream", On)
    before, calls = state(c, [0, 1]), len(host.seen.calls)
    with pytest.raises(UnsupportedError):
        go(given)
    assert state(c, [0, 1]) == before and len(host.seen.calls) == calls and now == [current]


# -------------------------------------------------------------------- outputs --
@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("pool", [False, True])
def test_decode_refuses_an_output_that_is_not_like_q(host, monkeypatch, pool, weighted):
    """Smaller, of another type, or strided: the kernel writes [batch, q_heads, 128] adjacent floats."""
    if pool:
        c = host(8)
        rids = [fill(c, 40), fill(c, 33)]
        go = lambda q, **k: c.flash_decode(0, rids, q, **k)  # noqa: E731
    else:
        c = ring(host)
        monkeypatch.setattr(kv.Kv3Cache, "__len__", lambda self: 40)
        go = c.flash_decode
    q = torch.zeros((2, 4, 128))
    more = {"weights": torch.zeros((2, 2, 40))} if weighted else {}
    out = torch.empty_like(q)
    assert go(q, out=out, **more) is out and go(q, **more).shape == q.shape
    calls = len(host.seen.calls)
    for bad in (torch.zeros((2, 4, 64)), torch.zeros((1, 4, 128)), q.double(), q.bfloat16(), [0.0],
                torch.zeros((2, 4, 256))[:, :, :128], torch.zeros((4, 2, 128)).transpose(0, 1)):
        with pytest.raises(ShapeError):
            go(q, out=bad, **more)
    assert len(host.seen.calls) == calls
