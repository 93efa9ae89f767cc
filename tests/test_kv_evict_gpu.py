"""Accumulated attention weight, eviction by it, and keeping chosen positions of the 3-bit cache.

Weights: the decode's scores are off by at most 2^-20 of 3 X, X = scale * sum|q| * max|k| (its q has
31 bits, the sums are fp32); exp2 and 1 / l add (n / 32 + 32) 2^-24; a sum over G heads and the addition to the
running weight a few 2^-24.  So |w - exact| <= exact * (2 * 3 X 2^-20 + (n / 32 + 64) 2^-24).  Selection and moves
are exact.
"""
import ctypes as C

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

D = 128


@pytest.fixture(scope="module")
def kv():
    assert torch.cuda.is_available()
    from ferrisres_b200 import kv as m
    return m


@pytest.fixture(scope="module")
def paged():
    from ferrisres_b200 import paged as m
    return m


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def rand(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def probs(q, k):
    """(p summed over each group [H, n], X) in 64 bits: q [Hq, D], k [n, H, D]."""
    n, H, _ = k.shape
    G = q.shape[0] // H
    out = torch.zeros((H, n), dtype=torch.float64, device="cuda")
    X = 0.0
    for h in range(q.shape[0]):
        kk = k[:, h // G].double()
        out[h // G] += torch.softmax(kk @ q[h].double() / D ** 0.5, 0)
        X = max(X, float(q[h].abs().sum() * kk.abs().max()) / D ** 0.5)
    return out, X


def check_weights(got, before, p, X, n):
    exact = before.double() + p
    tol = exact * (6 * X * 2.0 ** -20 + (n / 32 + 64) * 2.0 ** -24)
    assert bool(((got.double() - exact).abs() <= tol).all())


@pytest.mark.parametrize("mode", ["R", "T"])
@pytest.mark.parametrize("case", [(1, 1, 1, 1), (2, 31, 8, 2), (1, 32, 4, 4), (3, 700, 14, 2), (1, 1025, 40, 8),
                                  (2, 5000, 32, 8), (1, 20000, 5, 1)])
def test_weights(kv, case, mode):
    B, n, Hq, H = case
    g = generator(n)
    c = kv.Kv3Cache(B, H, n, mode=mode, seed=2)
    c.append(rand(g, B, n, H, D), rand(g, B, n, H, D))
    q = 2 * rand(g, B, Hq, D)
    w = torch.rand((B, H, n + 5), generator=g, device="cuda") / n
    w0 = w.clone()
    out = c.flash_decode(q, weights=w)
    assert torch.equal(out, c.flash_decode(q))  # the same kernel, the same bits
    assert torch.equal(w[:, :, n:], w0[:, :, n:])  # behind the last position: left alone
    k, _ = c.get_range(0, n)
    for b in range(B):
        p, X = probs(q[b], k[b])
        # mode T's keys are rotated back in fp32 for this comparison: 2^-17 of the scores
        check_weights(w[b, :, :n], w0[b, :, :n], p, X * (1 if mode == "R" else 4), n)
    c.ctx.check()
    c.close()


def test_decode_repeats_bit_for_bit(kv):
    """The warps of a split merge in the stage buffers: none may write there while a slower one
    still reads its block.  Short splits make the warps end far apart."""
    g = generator(20)
    for n in (1000, 8190):
        c = kv.Kv3Cache(4, 8, n)
        x = rand(g, 4, n, 8, D)
        c.append(x, x)
        q = rand(g, 4, 32, D)
        ref = c.flash_decode(q)
        for _ in range(300):
            assert torch.equal(c.flash_decode(q), ref)
        c.close()


def test_weights_in_strided_rows_and_moved_ring(kv):
    g = generator(3)
    c = kv.Kv3Cache(2, 2, 128)
    c.append(rand(g, 2, 120, 2, D), rand(g, 2, 120, 2, D))
    c.evict_front(45)
    c.append(rand(g, 2, 50, 2, D), rand(g, 2, 50, 2, D))
    n = len(c)
    big = torch.zeros((2, 2, 300), device="cuda")
    q = rand(g, 2, 6, D)
    side = torch.cuda.Stream()
    c.flash_decode(q, weights=big[:, :, 3:3 + n], stream=side)
    side.synchronize()
    k, _ = c.get_range(0, n)
    for b in range(2):
        p, X = probs(q[b], k[b])
        check_weights(big[b, :, 3:3 + n], torch.zeros_like(p), p, X, n)
    assert float(big[:, :, :3].abs().max()) == 0 and float(big[:, :, 3 + n:].abs().max()) == 0
    c.close()


def test_weights_paged(paged):
    g = generator(4)
    lens = [1, 40, 0, 333]
    c = paged.PagedKv3Cache(1, 40, 2)
    rids = [c.create_request() for _ in lens]
    for r, n in zip(rids, lens):
        if n:
            c.append(0, [r], rand(g, 1, n, 2, D), rand(g, 1, n, 2, D))
    q = rand(g, 4, 8, D)
    w = torch.zeros((4, 2, 340), device="cuda")
    out = c.flash_decode(0, rids, q, weights=w)
    assert torch.equal(out, c.flash_decode(0, rids, q))
    for i, (r, n) in enumerate(zip(rids, lens)):
        assert float(w[i, :, n:].abs().max()) == 0
        if n:
            k, _ = c.get_range(0, [r], 0, n)
            p, X = probs(q[i], k[0])
            check_weights(w[i, :, :n], torch.zeros_like(p), p, X, n)
    c.ctx.check()
    c.close()


def select_plain(w, n, keep, recent):
    """Kept positions of one row, by a stable sort."""
    if n <= keep:
        return np.concatenate([np.arange(n), np.full(keep - n, -1)])
    x = w[:n - recent].astype(np.float64) + 0.0
    x[np.isnan(x)] = np.inf
    x = np.where(np.isnan(w[:n - recent]), np.float64(1e300), np.where(np.isinf(x), np.sign(x) * 1e200, x))
    order = np.argsort(-x, kind="stable")[:keep - recent]
    return np.concatenate([np.sort(order), np.arange(n - recent, n)])


def weights_of(kind, rng, shape):
    if kind == "lognormal":
        return np.exp(3 * rng.standard_normal(shape)).astype(np.float32)
    if kind == "ties":
        return rng.integers(0, 4, shape).astype(np.float32)
    if kind == "equal":
        return np.full(shape, 0.25, np.float32)
    w = rng.standard_normal(shape).astype(np.float32)
    w[..., ::7] = 0.0
    w[..., 3::11] = -0.0
    w[..., 5::13] = np.nan
    w[..., 2::17] = np.inf
    w[..., 1::19] = -np.inf
    w[..., 4::23] = 1e-42
    return w


@pytest.mark.parametrize("kind", ["lognormal", "ties", "equal", "special"])
@pytest.mark.parametrize("case", [(1, 1, 1, 1, 0), (2, 2, 5, 1, 0), (1, 3, 100, 100, 3), (1, 1, 100, 99, 99),
                                  (2, 8, 1000, 500, 100), (1, 1, 5000, 7, 0), (1, 2, 17000, 16384, 2000),
                                  (3, 1, 2049, 2048, 0), (1, 1, 300000, 1000, 10), (1, 1, 400000, 390001, 1)])
def test_select(kv, case, kind):
    B, H, n, keep, recent = case
    rng = np.random.default_rng(n + keep)
    w = weights_of(kind, rng, (B, H, n))
    idx, out = kv.select_heavy(torch.from_numpy(w).cuda(), keep, recent)
    idx, out = idx.cpu().numpy(), out.cpu().numpy()
    for b in range(B):
        for h in range(H):
            ref = select_plain(w[b, h], n, keep, recent)
            assert (idx[b, h] == ref).all()
            m = min(n, keep)
            assert (out[b, h, :m].view(np.uint32) == w[b, h, ref[:m]].view(np.uint32)).all()
            assert (out[b, h, m:] == 0).all()


def test_select_ragged_strided(kv):
    rng = np.random.default_rng(9)
    lens = [0, 1, 7, 8, 9, 500, 600]
    w = rng.random((len(lens), 2, 700)).astype(np.float32)
    t = torch.from_numpy(w).cuda()[:, :, :600]
    idx, out = kv.select_heavy(t, 8, 3, seq_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    assert out.shape == t.shape and out.is_contiguous()
    for b, n in enumerate(lens):
        for h in range(2):
            ref = select_plain(w[b, h], n, 8, min(3, n))
            assert (idx[b, h].cpu().numpy() == ref).all()
            m = min(n, 8)
            assert (out[b, h, :m].cpu().numpy() == w[b, h, ref[:m]]).all()
            assert float(out[b, h, m:].abs().max()) == 0
    # a length beyond the rows is reported and held within them
    from ferrisres_b200._lib import ShapeError
    from ferrisres_b200.gpu import get_context
    kv.select_heavy(t, 8, 3, seq_lens=torch.full((7,), 601, dtype=torch.int32, device="cuda"))
    with pytest.raises(ShapeError):
        get_context(t.device.index).check()
    for bad in ((0, 0), (8, 9), (8, -1)):
        with pytest.raises(ShapeError):
            kv.select_heavy(t, *bad)
    with pytest.raises(ShapeError):
        kv.select_heavy(t, 8, 0, length=601)


def stored(c, *a):
    return [t.cpu().numpy() for t in c.export_range(*a)]


def gather(store, idx, H):
    """Stored form of positions idx [B, H, n] of store (codes [B, S, H*48], mm [B, S, H, 2])."""
    out = []
    for t in store:
        B, S = t.shape[:2]
        x = t.reshape(B, S, H, -1)
        out.append(np.stack([np.stack([x[b, idx[b, h], h] for h in range(H)], 1) for b in range(B)]))
    return out


def assert_store(got, want):
    for a, b in zip(got, want):
        b = b.reshape(a.shape)
        assert a.dtype == b.dtype and (a.view(np.uint8) == b.view(np.uint8)).all()


def random_lists(rng, B, H, n, m):
    return np.stack([np.stack([np.sort(rng.choice(n, m, replace=False)) for _ in range(H)])
                     for _ in range(B)]).astype(np.int32)


@pytest.mark.parametrize("mode", ["R", "T"])
@pytest.mark.parametrize("case", [(1, 1, 1, 1, 0), (2, 3, 40, 13, 0), (1, 2, 700, 333, 70), (2, 1, 64, 32, 32),
                                  (1, 8, 5000, 4700, 0), (1, 1, 9000, 10, 0), (3, 2, 2500, 2500, 0),
                                  (1, 4, 300, 0, 17), (2, 70, 100, 50, 20)])
def test_keep(kv, case, mode):
    B, H, n, m, start = case
    rng, g = np.random.default_rng(n), generator(n)
    c = kv.Kv3Cache(B, H, n + 3, mode=mode)
    x = rand(g, B, n, H, D)
    c.append(x, x + rand(g, B, n, H, D))
    before = stored(c, 0, n)
    idx = start + random_lists(rng, B, H, n - start, m)
    c.keep(torch.from_numpy(idx).cuda(), start=start)
    assert len(c) == start + m
    if start + m:
        full = np.concatenate([np.broadcast_to(np.arange(start), (B, H, start)), idx], 2)
        assert_store(stored(c, 0, start + m), gather(before, full, H))
    # and the cache goes on from there
    y = rand(g, B, 2, H, D)
    c.append(y, y)
    k, _ = c.get_range(0, start + m + 2)
    assert k.shape[1] == start + m + 2
    c.ctx.check()
    c.close()


def test_keep_on_a_moved_ring(kv):
    """Heads inside a block, wraps, and a full ring whose last block is the head's own."""
    rng, g = np.random.default_rng(1), generator(1)
    B, H, cap = 2, 2, 256
    for drop, add, m, start in ((37, 37, 200, 0), (37, 37, 256, 0), (37, 37, 250, 3), (200, 199, 100, 100),
                                (33, 1, 224, 0), (64, 64, 256, 0), (37, 37, 12, 244)):
        c = kv.Kv3Cache(B, H, cap)
        c.append(rand(g, B, cap, H, D), rand(g, B, cap, H, D))
        c.evict_front(drop)
        c.append(rand(g, B, add, H, D), rand(g, B, add, H, D))
        n = len(c)
        before = stored(c, 0, n)
        idx = start + random_lists(rng, B, H, n - start, m)
        c.keep(torch.from_numpy(idx).cuda(), start=start)
        full = np.concatenate([np.broadcast_to(np.arange(start), (B, H, start)), idx], 2)
        assert_store(stored(c, 0, start + m), gather(before, full, H))
        c.ctx.check()
        c.close()


def test_keep_list_forms_and_refusals(kv):
    from ferrisres_b200._lib import ShapeError
    g = generator(2)
    B, H, n = 2, 3, 50
    c = kv.Kv3Cache(B, H, 64)

    def fill():
        c.reset()
        c.append(x, x)

    x = rand(g, B, n, H, D)
    fill()
    before = stored(c, 0, n)
    one = [1, 5, 5, 49]  # a position may be kept twice
    per = [[0, 7, 9, 11], [2, 3, 30, 49]]
    for idx, full in ((torch.tensor(one), np.broadcast_to(np.array(one), (B, H, 4))),
                      (torch.tensor(per, dtype=torch.int32),
                       np.broadcast_to(np.array(per)[:, None], (B, H, 4)))):
        fill()
        c.keep(idx.cuda())
        assert_store(stored(c, 0, 4), gather(before, np.ascontiguousarray(full), H))
    # entries that would overwrite a later source, or lie outside, are skipped and reported
    for bad in ([3, 0, 9, 10], [3, 4, 5, 50], [-1, 4, 5, 6], [2**40, 4, 5, 6]):
        fill()
        c.keep(torch.tensor(bad).cuda())
        with pytest.raises(ShapeError):
            c.ctx.check()
        want = [b if i <= b < n else i for i, b in enumerate(bad)]
        assert_store(stored(c, 0, 4), gather(before, np.broadcast_to(np.array(want), (B, H, 4)), H))
    fill()
    for idx, start in ((torch.zeros(51, dtype=torch.int32), 0), (torch.zeros(4, dtype=torch.int32), 47),
                       (torch.zeros(4, dtype=torch.int32), -1), (torch.zeros((3, 4), dtype=torch.int32), 0)):
        with pytest.raises(ShapeError):
            c.keep(idx.cuda(), start=start)
    assert len(c) == n
    c.ctx.check()
    c.close()


def test_keep_nothing_and_evict_nothing(kv):
    g = generator(40)
    c = kv.Kv3Cache(2, 2, 64)
    x = rand(g, 2, 40, 2, D)
    none = torch.empty((2, 2, 0), dtype=torch.int32, device="cuda")
    idx, w = c.evict_heavy(torch.zeros((2, 2, 8), device="cuda"), 4, 2)  # an empty cache
    assert bool((idx == -1).all()) and bool((w == 0).all()) and len(c) == 0
    idx, w = c.evict_heavy(torch.zeros((2, 2, 0), device="cuda"), 4, 2)
    assert bool((idx == -1).all()) and w.shape == (2, 2, 0)
    c.append(x, x)
    before = stored(c, 0, 40)
    c.keep(none, start=33)  # rejected drafts: the cache is cut
    assert len(c) == 33
    for a, b in zip(stored(c, 0, 33), before):
        assert (a == b[:, :33]).all()
    c.keep(none)
    assert len(c) == 0
    c.append(x, x)
    for a, b in zip(stored(c, 0, 40), before):
        assert (a == b).all()
    c.ctx.check()
    c.close()


@pytest.mark.parametrize("share", [0.97, 0.6, 0.2, 0.03])
def test_keep_shares(kv, share):
    """Sources that span few records, many, and far more than are staged at once."""
    rng, g = np.random.default_rng(int(100 * share)), generator(41)
    B, H, n = 2, 3, 6000
    c = kv.Kv3Cache(B, H, n)
    c.append(rand(g, B, n, H, D), rand(g, B, n, H, D))
    before = stored(c, 0, n)
    idx = random_lists(rng, B, H, n, int(n * share))
    c.keep(torch.from_numpy(idx).cuda())
    assert_store(stored(c, 0, idx.shape[2]), gather(before, idx, H))
    # not ascending, but no entry below its place
    m = idx.shape[2] // 2
    free = np.stack([np.stack([rng.integers(np.arange(m), idx.shape[2]) for _ in range(H)])
                     for _ in range(B)]).astype(np.int32)
    before = stored(c, 0, idx.shape[2])
    c.keep(torch.from_numpy(free).cuda())
    assert_store(stored(c, 0, m), gather(before, free, H))
    c.ctx.check()
    c.close()


def test_evict_heavy(kv):
    g, rng = generator(5), np.random.default_rng(5)
    B, H, n, keep, recent = 2, 2, 1000, 600, 64
    c = kv.Kv3Cache(B, H, n)
    c.append(rand(g, B, n, H, D), rand(g, B, n, H, D))
    before = stored(c, 0, n)
    w = torch.zeros((B, H, n), device="cuda")
    for _ in range(4):
        c.flash_decode(2 * rand(g, B, 8, D), weights=w)
    host = w.cpu().numpy()
    idx, w2 = c.evict_heavy(w, keep, recent)
    assert len(c) == keep and w2.shape == w.shape
    ref = np.stack([np.stack([select_plain(host[b, h], n, keep, recent) for h in range(H)]) for b in range(B)])
    assert (idx.cpu().numpy() == ref).all()
    assert_store(stored(c, 0, keep), gather(before, ref, H))
    # nothing to evict: the cache and the weights stay as they are
    idx, w3 = c.evict_heavy(w2, keep + 10, recent)
    assert len(c) == keep and torch.equal(w3[:, :, :keep], w2[:, :, :keep])
    assert bool((idx[:, :, keep:] == -1).all())
    out = c.flash_decode(rand(g, B, 8, D), weights=w3)
    assert bool(torch.isfinite(out).all())
    c.ctx.check()
    c.close()


def test_paged_keep_and_evict(paged):
    rng, g = np.random.default_rng(6), generator(6)
    H, lens = 2, [300, 5, 64, 97]
    c = paged.PagedKv3Cache(2, 40, H)
    rids = [c.create_request() for _ in lens]
    for r, n in zip(rids, lens):
        for layer in range(2):
            x = rand(g, 1, n, H, D)
            c.append(layer, [r], x, -x)
    before = [stored(c, 0, [r], 0, n) for r, n in zip(rids, lens)]
    other = [stored(c, 1, [r], 0, n) for r, n in zip(rids, lens)]
    w = torch.from_numpy(rng.random((4, H, 300)).astype(np.float32)).cuda()
    idx, w2 = c.evict_heavy(0, rids, w, 64, 10)
    free = c.manager.num_free_blocks()
    assert [c.seq_len(r, 0) for r in rids] == [64, 5, 64, 64]
    assert [c.seq_len(r, 1) for r in rids] == lens
    assert [len(c.block_table(r, 0)) for r in rids] == [2, 1, 2, 2]
    assert free == 40 - (2 + 1 + 2 + 2) - (10 + 1 + 2 + 4)
    for i, (r, n) in enumerate(zip(rids, lens)):
        ref = np.stack([select_plain(w[i, h].cpu().numpy(), n, 64, min(10, n)) for h in range(H)])
        assert (idx[i].cpu().numpy() == ref).all()
        m = min(n, 64)
        assert_store(stored(c, 0, [r], 0, m), gather(before[i], ref[None, :, :m], H))
        assert_store(stored(c, 1, [r], 0, n), other[i])
    # accepted paths of different lengths, from different starts
    c.keep(1, rids, torch.tensor([[290, 295, 299], [4, 4, 4], [1, 2, 3], [60, 70, 80]]).cuda(),
           counts=[3, 1, 0, 2], starts=[290, 4, 30, 20])
    assert [c.seq_len(r, 1) for r in rids] == [293, 5, 30, 22]
    for i, full in enumerate(([*range(290), 290, 295, 299], range(5), range(30), [*range(20), 60, 70])):
        full = np.broadcast_to(np.array(list(full)), (1, H, len(full)))
        assert_store(stored(c, 1, [rids[i]], 0, full.shape[2]), gather(other[i], full, H))
    c.ctx.check()
    for r in rids:
        c.free_request(r)
    assert c.manager.num_free_blocks() == 40
    c.close()


def test_paged_keep_spares_a_fork(paged):
    from ferrisres_b200._lib import OOMError, ShapeError
    g = generator(7)
    H = 2
    c = paged.PagedKv3Cache(1, 10, H)
    a = c.create_request()
    x = rand(g, 1, 100, H, D)
    c.append(0, [a], x, -x)
    b = c.fork_request(a)
    before = stored(c, 0, [a], 0, 100)
    idx = torch.tensor([40, 50, 99], dtype=torch.int32, device="cuda")
    c.keep(0, [a, b], idx, starts=[33, 33], counts=[3, 2])
    for r, full in ((a, [*range(33), 40, 50, 99]), (b, [*range(33), 40, 50])):
        full = np.broadcast_to(np.array(full), (1, H, len(full)))
        assert_store(stored(c, 0, [r], 0, full.shape[2]), gather(before, full, H))
    ta, tb = c.block_table(a), c.block_table(b)
    assert ta[0] == tb[0] and ta[1] != tb[1] and len(ta) == len(tb) == 2
    assert c.manager.num_free_blocks() == 7
    with pytest.raises(ShapeError):
        c.keep(0, [a, a], idx[:1])
    with pytest.raises(ShapeError):
        c.keep(0, [a], idx, counts=[4])
    with pytest.raises(ShapeError):
        c.keep(0, [a], idx, starts=[34])
    # no page for the copy: nothing changes
    d = c.fork_request(a)
    e = c.create_request()
    c.append(0, [e], rand(g, 1, 7 * 32, H, D), rand(g, 1, 7 * 32, H, D))
    with pytest.raises(OOMError):
        c.keep(0, [d], torch.tensor([5], dtype=torch.int32, device="cuda"))
    assert c.seq_len(d) == 36 and c.block_table(d) == c.block_table(a)
    c.ctx.check()
    c.close()


def test_paged_entry_reports_bad_rows(paged):
    """Lengths, counts and pages that do not fit are skipped and reported; the rest is moved."""
    from ferrisres_b200._lib import ShapeError, call
    from ferrisres_b200.gpu import _dptr, _stream_ptr
    g = generator(8)
    c = paged.PagedKv3Cache(1, 4, 1)
    a, b = c.create_request(), c.create_request()
    x = rand(g, 2, 40, 1, D)
    c.append(0, [a, b], x, x)
    idx = torch.tensor([[35, 36], [35, 36]], dtype=torch.int32, device="cuda")
    good = torch.tensor([c.block_table(a), c.block_table(b)], dtype=torch.int32, device="cuda")
    before = stored(c, 0, [a], 0, 40)

    def go(tables, lens, starts, counts):
        t = [torch.tensor(v, dtype=torch.int32, device="cuda") for v in (lens, starts, counts)]
        call("ft_kvp_keep", c.ctx.handle, c.handle, 2, _dptr(tables), 2, _dptr(t[0]), _dptr(t[1]), _dptr(t[2]), 2,
             _dptr(idx), 2, 0, _stream_ptr())
        with pytest.raises(ShapeError):
            c.ctx.check()

    go(good, [65, 40], [0, 39], [2, 2])
    go(good, [-1, 40], [0, -1], [1, 1])
    go(good, [40, 40], [0, 0], [3, -2])
    assert_store(stored(c, 0, [a], 0, 40), before)
    bad = good.clone()
    bad[:, 1] = 4
    go(bad, [40, 40], [0, 0], [2, 2])  # the sources' page is unknown: the slots keep what they hold
    assert_store(stored(c, 0, [a], 0, 40), before)
    c.ctx.check()
    c.close()


def test_a_serving_loop(kv):
    """Drafts, verification, commit, decode with weights and eviction, step by step, against a cache
    that holds the same positions by plain appends."""
    g, rng = generator(9), np.random.default_rng(9)
    B, H, Hq, budget = 2, 2, 4, 200
    c = kv.Kv3Cache(B, H, 256)
    x = rand(g, B, 190, H, D)
    y = rand(g, B, 190, H, D)
    c.append(x, y)
    codes = [t.clone() for t in c.export_range(0, 190)]
    w = torch.zeros((B, H, 256), device="cuda")
    for step in range(6):
        T = int(rng.integers(2, 9))
        parents = [-1] + [int(rng.integers(-1, i)) for i in range(1, T)]
        P = len(c)
        c.append(rand(g, B, T, H, D), rand(g, B, T, H, D))
        drafts = c.export_range(P, P + T)
        c.tree_decode(rand(g, B, T, Hq, D), kv.tree_mask(parents))
        path = [T - 1]
        while parents[path[0]] >= 0:
            path.insert(0, parents[path[0]])
        c.keep(torch.tensor(path, device="cuda") + P, start=P)
        codes = [torch.cat([a, d[:, path]], 1) for a, d in zip(codes, drafts)]
        q = rand(g, B, Hq, D)
        out = c.flash_decode(q, weights=w)
        twin = kv.Kv3Cache(B, H, 512)
        twin.append_packed(*codes)
        assert torch.equal(twin.flash_decode(q), out)
        twin.close()
        if len(c) > budget:
            n = len(c)
            idx, w = c.evict_heavy(w, budget, 16)
            at = idx.long().transpose(1, 2)[..., None]
            codes = [torch.gather(t.reshape(B, n, H, -1), 1,
                                  at.expand(-1, -1, -1, t.reshape(B, n, H, -1).shape[-1])).reshape(
                                      (B, budget) + tuple(t.shape[2:])) for t in codes]
    assert len(c) <= budget + 8
    c.ctx.check()
    c.close()


def test_captured_keep_and_select(kv):
    g = generator(10)
    B, H, n = 1, 2, 400
    x = rand(g, B, n, H, D)
    c, d = kv.Kv3Cache(B, H, n), kv.Kv3Cache(B, H, n)
    c.append(x, x)
    d.append(x, x)
    w = torch.rand((B, H, n), generator=g, device="cuda")
    idx, _ = kv.select_heavy(w, 100, 10)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        i2, w2 = kv.select_heavy(w, 100, 10)
        c._keep(i2, 100, H * 100, 100, 0, None)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(i2, idx) and len(c) == 100
    d.keep(idx)
    assert_store(stored(c, 0, 100), stored(d, 0, 100))
    c.ctx.check()
    c.close()
    d.close()


@pytest.mark.parametrize("H", [1, 3, 8])
def test_packed_append_in_pieces(kv, paged, H):
    """Stored positions appended in pieces that begin and end inside blocks, from aligned and
    unaligned memory, read back byte for byte."""
    g, rng = generator(30 + H), np.random.default_rng(H)
    B, n = 2, 333
    src = kv.Kv3Cache(B, H, n)
    src.append(rand(g, B, n, H, D), rand(g, B, n, H, D))
    want = src.export_range(0, n)
    c = kv.Kv3Cache(B, H, 352)
    c.append(rand(g, B, 45, H, D), rand(g, B, 45, H, D))
    c.evict_front(45)  # the head lies inside a block, and the ring wraps
    p = paged.PagedKv3Cache(1, 30, H)
    rids = [p.create_request() for _ in range(B)]
    at = 0
    for m in (1, 30, 2, 64, 95, 7, 134):
        part = [t[:, at:at + m] for t in want]
        c.append_packed(*part)
        p.append_packed(0, rids, *part)
        at += m
    assert at == n
    for a, b in ((0, n), (1, 2), (31, 33), (40, 300), (332, 333)):
        for got in (c.export_range(a, b), p.export_range(0, rids, a, b)):
            for x, y in zip(got, want):
                assert torch.equal(x, y[:, a:b])
    # unaligned code bytes in and out
    from ferrisres_b200._lib import call
    from ferrisres_b200.gpu import _dptr, _stream_ptr
    c.reset()
    moved = []
    for t in (want[0], want[2]):
        raw = torch.zeros(t.numel() + 3, dtype=torch.uint8, device="cuda")
        raw[3:] = t.flatten()
        moved.append(raw)
    call("ft_kv3_append_packed", c.ctx.handle, c.handle, n, C.c_void_p(moved[0].data_ptr() + 3), _dptr(want[1]),
         C.c_void_p(moved[1].data_ptr() + 3), _dptr(want[3]), _stream_ptr())
    for raw in moved:
        raw.fill_(255)
    mm = [torch.empty_like(want[1]), torch.empty_like(want[3])]
    call("ft_kv3_export_range", c.ctx.handle, c.handle, 0, n, C.c_void_p(moved[0].data_ptr() + 3), _dptr(mm[0]),
         C.c_void_p(moved[1].data_ptr() + 3), _dptr(mm[1]), _stream_ptr())
    for raw, t in zip(moved, (want[0], want[2])):
        assert torch.equal(raw[3:], t.flatten()) and raw[:3].tolist() == [255] * 3
    assert torch.equal(mm[0], want[1]) and torch.equal(mm[1], want[3])
    p.ctx.check()
    for x in (src, c, p):
        x.close()
