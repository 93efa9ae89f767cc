"""Tree decode over the 3-bit cache against attention in 64 bits over the stored values.

Error bound, per output of a row.  Let X = scale * max_s sum_d |q_d| * max_d |k_sd| over the
positions that the row sees and V = max |v| over them; n of them.
  scores: q.k = min * sum(q) + step * sum(q c); |min| sum|q| <= X/scale and step * c <= 2 max|k|, so
    the parts add up to at most 3 X.  fp32 q enters as fp16 hi + lo, each rounded by half a step of
    2^-11 relative: 2^-22 of q; the products' fp32 sums, step and the two factors add a few 2^-24.
    Together 3 X 2^-20.  A bf16 q is exact in hi (mode R); rotated (mode T) it is rounded to fp16 by
    2^-11: 3 X 2^-11.
  weights: p is off by 2 x that (numerator and denominator) and a few 2^-22 of exp2; w enters as
    fp16 hi + lo: 2^-22, or hi alone: 2^-11, of terms that add up to at most 2 V.
  sums: n / 32 block sums added in fp32: (n / 32 + 16) 2^-24 of terms of at most 3 V.
  as a whole: these roundings are independent, so the 2-norm of an fp32 result's error stays well under the
    worst case: within 1e-5 of the result's (mode R, where the comparison's input is exact), the bound of the
    single-token decode.
  output: bf16 rounds by 2^-8 of the value, uniformly up to that, so by at most 2^-8 / sqrt(3) in the
    2-norm; what comes before (2^-11) hides in that: 0.6 * 2^-8 of the result's norm.
  mode T: the stored vectors rotated back in fp32 (the comparison's input) are off by about
    10 * 2^-24 of their norm <= 12 max|v|: 2^-17 V, and of k likewise: X 2^-17.
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


def rand(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def rand_mask(gen, B, T):
    """Random words, not only trees; draft 0 sees nothing of the drafts, draft 1 everything."""
    bits = torch.rand((B, T, T), generator=gen, device="cuda") < 0.5
    bits[:, 0] = False
    if T > 1:
        bits[:, 1] = True
    place = torch.arange(T, device="cuda", dtype=torch.int64)
    return (bits.long() << place).sum(-1), bits


def causal_bits(B, T):
    return torch.ones((T, T), dtype=torch.bool, device="cuda").tril().expand(B, T, T)


def exact(q, k, v, bits, scale=None):
    """(out, X, V) in 64 bits: q [T, Hq, D], k, v [n, H, D] as stored, bits [T, T]."""
    T, Hq, _ = q.shape
    n, H, _ = k.shape
    G = Hq // H
    scale = D ** -0.5 if scale is None else scale
    q, k, v = q.double(), k.double(), v.double()
    sees = torch.ones((T, n), dtype=torch.bool, device=q.device)
    sees[:, max(0, n - T):] = bits[:, max(0, T - n):]
    out, X, V = (torch.zeros((T, Hq, D), dtype=torch.float64, device=q.device) for _ in range(3))
    for h in range(Hq):
        x = scale * (q[:, h] @ k[:, h // G].T)
        x = x.masked_fill(~sees, -np.inf)
        top = x.amax(1, keepdim=True)
        p = torch.exp(x - torch.where(torch.isinf(top), 0.0, top))
        total = p.sum(1, keepdim=True)
        p = torch.where(total > 0, p / total, 0.0)
        vs = torch.where(sees[:, :, None].any(0), v[:, h // G], 0.0)
        out[:, h] = p @ vs
        ka = (k[:, h // G].abs().amax(1)[None] * sees).amax(1)
        va = (v[:, h // G].abs().amax(1)[None] * sees).amax(1)
        X[:, h] = (scale * q[:, h].abs().sum(1) * ka)[:, None]
        V[:, h] = va[:, None]
    return out, X, V


def check(got, ref, dtype, mode, n):
    out, X, V = ref
    bf16 = dtype == torch.bfloat16
    ds = 3 * X * (2.0 ** -11 if bf16 and mode == "T" else 2.0 ** -20)
    tol = V * (2 * ds + 2.0 ** -18 + 2 * (2.0 ** -11 if bf16 else 2.0 ** -22) + 3 * (n / 32 + 16) * 2.0 ** -24)
    if mode == "T":
        tol = tol + V * (2.0 ** -17 + 2 * X * 2.0 ** -17)
    if bf16:
        tol = tol + 2.0 ** -8 * out.abs()
    err = (got.double() - out).abs()
    bad = err > tol
    assert not bad.any(), f"{int(bad.sum())} off, worst {float((err / tol.clamp_min(1e-300)).max()):.2f} of the bound"
    if not bf16 and mode == "R":
        assert float(err.norm()) <= 1e-5 * float(out.norm()), float(err.norm() / out.norm())


CASES = [
    # B, n, T, Hq, H
    (1, 1, 1, 1, 1), (1, 5, 5, 8, 2), (2, 31, 3, 4, 4), (1, 32, 32, 2, 1), (2, 33, 8, 8, 2),
    (1, 64, 64, 4, 2), (3, 127, 16, 14, 2), (1, 129, 1, 40, 8), (2, 517, 5, 8, 2), (1, 700, 64, 16, 1),
    (2, 1000, 21, 15, 3), (1, 4099, 8, 32, 8), (1, 2500, 63, 10, 2), (5, 300, 7, 7, 7),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mode", ["R", "T"])
@pytest.mark.parametrize("case", CASES)
def test_ring_tree_decode(kv, case, mode, dtype):
    B, n, T, Hq, H = case
    g = generator(n * T + Hq)
    c = kv.Kv3Cache(B, H, n, mode=mode, seed=3)
    c.append(rand(g, B, n, H, D), rand(g, B, n, H, D))
    q = (2 * rand(g, B, T, Hq, D)).to(dtype)
    mask, bits = rand_mask(g, B, T)
    out = c.tree_decode(q, mask)
    k, v = c.get_range(0, n)
    for b in range(B):
        check(out[b], exact(q[b], k[b], v[b], bits[b]), dtype, mode, n)
    # without a mask: draft i sees drafts 0..i
    out = c.tree_decode(q)
    for b in range(B):
        check(out[b], exact(q[b], k[b], v[b], causal_bits(B, T)[b]), dtype, mode, n)
    c.ctx.check()
    c.close()


@pytest.mark.parametrize("mode", ["R", "T"])
@pytest.mark.parametrize("case", [(1, 128 + 1, 1, 1, 1), (1, 256 + 3, 2, 8, 2), (2, 385, 1, 16, 2), (1, 1100, 4, 32, 8),
                                  (1, 2100, 64, 2, 1), (2, 1500, 64, 4, 1), (1, 3000, 33, 20, 4), (3, 900, 64, 15, 3),
                                  (1, 20000, 8, 8, 2), (8, 640, 17, 8, 8)])
def test_whole_prefix_tiles(kv, case, mode):
    """bf16 queries: the 128-position tiles in front of the drafts, one and many, few and many rows."""
    B, n, T, Hq, H = case
    g = generator(n + T)
    c = kv.Kv3Cache(B, H, n, mode=mode, seed=3)
    spread = 0.2 + 2 * torch.rand((H, D), generator=g, device="cuda")
    c.append(rand(g, B, n, H, D) * spread, rand(g, B, n, H, D) * spread)
    q = (2 * rand(g, B, T, Hq, D)).bfloat16()
    mask, bits = rand_mask(g, B, T)
    out = c.tree_decode(q, mask)
    c.ctx.check()
    k, v = c.get_range(0, n)
    for b in range(B):
        check(out[b], exact(q[b], k[b], v[b], bits[b]), torch.bfloat16, mode, n)
    c.close()


def test_scores_that_rise(kv):
    """Maxima that move by a little and by a lot along the sequence, values that grow by 2^20, constant
    vectors: the references of the prefix tiles move in every way."""
    g = generator(21)
    n, T, Hq, H = 2500, 6, 8, 2
    for kind in ("rise", "fall", "steps", "huge", "values", "constant"):
        k, v = rand(g, 1, n, H, D), rand(g, 1, n, H, D)
        q = (2 * rand(g, 1, T, Hq, D)).bfloat16()
        at = torch.arange(n, device="cuda")[None, :, None, None]
        along = torch.nn.functional.normalize(q.float().mean((1, 2)), dim=-1)  # moves every row's score
        if kind == "rise":
            k = k + along * at * 0.03
        elif kind == "fall":
            k = k - along * at * 0.03
        elif kind == "steps":
            k = k + along * (at // 300 * 37 % 90)
        elif kind == "huge":
            k = k * 40
        elif kind == "values":
            v = v * torch.exp2(torch.div(at, 128, rounding_mode="floor").float())
        else:
            v[:, ::2] = 0.5
            v[:, 1200:1600] = 0.0
            k[:, 700] = 1.0
        c = kv.Kv3Cache(1, H, n)
        c.append(k, v)
        out = c.tree_decode(q)
        c.ctx.check()
        kk, vv = c.get_range(0, n)
        check(out[0], exact(q[0], kk[0], vv[0], causal_bits(1, T)[0]), torch.bfloat16, "R", n)
        c.close()


def test_moved_ring(kv):
    """Heads that start inside a block, and a ring that wraps onto its first block."""
    g = generator(5)
    B, H, Hq, T = 2, 2, 6, 9
    c = kv.Kv3Cache(B, H, 256)
    c.append(rand(g, B, 250, H, D), rand(g, B, 250, H, D))
    for drop, add in ((7, 13), (100, 95), (31, 31), (33, 38)):
        q16 = (2 * rand(g, B, T, Hq, D)).bfloat16()
        mask, bits = rand_mask(g, B, T)
        out = c.tree_decode(q16, mask)  # heads inside a block: its slots are the edges' work
        k, v = c.get_range(0, len(c))
        for b in range(B):
            check(out[b], exact(q16[b], k[b], v[b], bits[b]), torch.bfloat16, "R", len(c))
        c.evict_front(drop)
        c.append(rand(g, B, add, H, D), rand(g, B, add, H, D))
        n = len(c)
        assert c.capacity == 256
        q = rand(g, B, T, Hq, D)
        mask, bits = rand_mask(g, B, T)
        out = c.tree_decode(q, mask)
        k, v = c.get_range(0, n)
        for b in range(B):
            check(out[b], exact(q[b], k[b], v[b], bits[b]), torch.float32, "R", n)
    assert n == 256  # full: the last block of the sequence shares the head's
    c.ctx.check()
    c.close()


def test_shared_mask_scale_out_and_stream(kv):
    g = generator(6)
    c = kv.Kv3Cache(2, 2, 100)
    c.append(rand(g, 2, 90, 2, D), rand(g, 2, 90, 2, D))
    q = rand(g, 2, 4, 4, D)
    tree = kv.tree_mask([-1, 0, 0, 1])
    a = c.tree_decode(q, tree, scale=0.3)
    k, v = c.get_range(0, 90)
    bits = torch.tensor([[1, 0, 0, 0], [1, 1, 0, 0], [1, 0, 1, 0], [1, 1, 0, 1]], dtype=torch.bool, device="cuda")
    check(a[0], exact(q[0], k[0], v[0], bits, 0.3), torch.float32, "R", 90)
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    assert c.tree_decode(q, tree.expand(2, 4), scale=0.3, out=out, stream=side) is out
    side.synchronize()
    assert torch.equal(out, a)
    # strided queries are the same queries
    wide = torch.zeros((2, 4, 8, D), device="cuda")
    wide[:, :, ::2] = q
    assert torch.equal(c.tree_decode(wide[:, :, ::2], tree, scale=0.3), a)
    c.close()


def test_one_draft_is_the_decode(kv):
    """T = 1 without a mask is the single-token decode, to both kernels' bounds."""
    g = generator(7)
    c = kv.Kv3Cache(2, 2, 300)
    c.append(rand(g, 2, 300, 2, D), rand(g, 2, 300, 2, D))
    q = rand(g, 2, 1, 8, D)
    a, b = c.tree_decode(q)[:, 0].double(), c.flash_decode(q[:, 0].contiguous()).double()
    assert float((a - b).abs().max()) <= 2e-5
    c.close()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_places_do_not_matter(kv, dtype):
    """Drafts that a row does not see may hold infinities, NaN or huge values."""
    g = generator(8)
    B, P, T, H, Hq = 1, 70, 12, 2, 8
    k, v = rand(g, B, P + T, H, D), rand(g, B, P + T, H, D)
    outs = []
    for fill in (0.0, float("inf"), float("-inf"), float("nan"), 1e30, -3e38):
        c = kv.Kv3Cache(B, H, P + T)
        kk, vv = k.clone(), v.clone()
        kk[:, P + 6:, :, ::3] = fill
        vv[:, P + 6:, :, 1::3] = fill
        c.append(kk, vv)
        q = (2 * rand(generator(9), B, T, Hq, D)).to(dtype)
        mask = torch.tensor([(2 << i) - 1 for i in range(T)], device="cuda") & 63  # none of 6..11
        outs.append(c.tree_decode(q, mask))
        assert bool(torch.isfinite(outs[-1].float()).all())
        c.close()
    for o in outs[1:]:
        assert torch.equal(o, outs[0])


def test_bad_query_rows_stay_alone(kv):
    g = generator(10)
    c = kv.Kv3Cache(1, 2, 200)
    c.append(rand(g, 1, 200, 2, D), rand(g, 1, 200, 2, D))
    q = rand(g, 1, 6, 8, D)
    ref = c.tree_decode(q)
    for bad in (float("nan"), float("inf"), float("-inf")):
        z = q.clone()
        z[0, 2, 5, 17] = bad
        out = c.tree_decode(z)
        assert bool(torch.isnan(out[0, 2, 5]).all())
        out[0, 2, 5] = ref[0, 2, 5]
        assert torch.equal(out, ref)
    # rows of very different sizes, subnormal and zero ones among them
    z = q * torch.tensor([1e-42, 1e-30, 0.0, 1.0, 30.0, 1e3], device="cuda")[None, :, None, None]
    out = c.tree_decode(z)
    k, v = c.get_range(0, 200)
    check(out[0], exact(z[0], k[0], v[0], causal_bits(1, 6)[0]), torch.float32, "R", 200)
    c.close()


def test_values_of_any_size(kv):
    """K and V far from 1: the codes enter as they are, so nothing overflows in 16 bits."""
    g = generator(11)
    for size in (1e-20, 1e-6, 1e5, 1e20):
        c = kv.Kv3Cache(1, 1, 200)
        c.append(rand(g, 1, 200, 1, D) * size, rand(g, 1, 200, 1, D) * size)
        q = rand(g, 1, 3, 2, D) / size
        k, v = c.get_range(0, 200)
        check(c.tree_decode(q)[0], exact(q[0], k[0], v[0], causal_bits(1, 3)[0]), torch.float32, "R", 200)
        c.close()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mode", ["R", "T"])
def test_paged_tree_decode(paged, mode, dtype):
    g = generator(12)
    H, Hq, T, lens = 2, 10, 11, [11, 45, 100, 257, 1030]
    c = paged.PagedKv3Cache(2, 80, H, mode=mode, seed=4)
    rids = [c.create_request() for _ in lens]
    for r, n in zip(rids, lens):
        for part in (n // 2, n - n // 2):
            c.append(1, [r], rand(g, 1, part, H, D), rand(g, 1, part, H, D))
    q = (2 * rand(g, len(lens), T, Hq, D)).to(dtype)
    mask, bits = rand_mask(g, len(lens), T)
    out = c.tree_decode(1, rids, q, mask)
    for i, (r, n) in enumerate(zip(rids, lens)):
        k, v = c.get_range(1, [r], 0, n)
        check(out[i], exact(q[i], k[0], v[0], bits[i]), dtype, mode, n)
    c.ctx.check()
    c.close()


def test_short_empty_and_bad_sequences(paged):
    """The C entry: sequences shorter than the drafts, empty ones, and bad pages and lengths."""
    from ferrisres_b200._lib import ShapeError, call
    from ferrisres_b200.gpu import _dptr, _stream_ptr
    g = generator(13)
    c = paged.PagedKv3Cache(1, 8, 1)
    r = c.create_request()
    c.append(0, [r], rand(g, 1, 40, 1, D), rand(g, 1, 40, 1, D))
    tables = torch.tensor([c.block_table(r)] * 3, dtype=torch.int32, device="cuda")
    lens = torch.tensor([3, 0, 40], dtype=torch.int32, device="cuda")
    T = 5
    q = rand(g, 3, T, 2, D)
    out = torch.full_like(q, 7.0)

    def go(tables, lens):
        call("ft_kvp_tree_decode", c.ctx.handle, c.handle, 3, _dptr(tables), 2, _dptr(lens), 40, 0, T,
             _dptr(q), 0, 2, None, C.c_float(0.0), _dptr(out), _stream_ptr())

    go(tables, lens)
    c.ctx.check()
    k, v = c.get_range(0, [r], 0, 40)
    assert bool((out[1] == 0).all()) and bool((out[0, :2] == 0).all())  # drafts 0, 1 see nothing
    for b, n in ((0, 3), (2, 40)):
        check(out[b], exact(q[b], k[0, :n], v[0, :n], causal_bits(1, T)[0]), torch.float32, "R", n)
    for bad_t, bad_l in ((99, 40), (-1, 40), (0, 41), (0, -1)):
        t, l = tables.clone(), lens.clone()
        t[2, 1] = bad_t
        l[2] = bad_l
        go(t, l)
        if bad_t:
            with pytest.raises(ShapeError):
                c.ctx.check()
        elif bad_l in (41, -1):
            with pytest.raises(ShapeError):
                c.ctx.check()
    c.ctx.check()
    c.close()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_two_streams_and_a_graph(kv, dtype):
    """Caches of their own on streams of their own, one call captured: results as one by one."""
    g = generator(30)
    caches, qs, refs = [], [], []
    for i, n in enumerate((900, 2600)):
        c = kv.Kv3Cache(2, 2, n)
        c.append(rand(g, 2, n, 2, D), rand(g, 2, n, 2, D))
        caches.append(c)
        qs.append((2 * rand(g, 2, 40, 8, D)).to(dtype))
        refs.append(c.tree_decode(qs[i]))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    out = torch.empty_like(qs[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        caches[0].tree_decode(qs[0], out=out)
    for _ in range(20):
        with torch.cuda.stream(streams[0]):
            graph.replay()
        got = caches[1].tree_decode(qs[1], stream=streams[1])
    torch.cuda.synchronize()
    assert torch.equal(out, refs[0]) and torch.equal(got, refs[1])
    for c in caches:
        c.ctx.check()
        c.close()


def test_refusals(kv, paged):
    from ferrisres_b200._lib import ShapeError, UnsupportedError
    c = kv.Kv3Cache(1, 2, 64)
    q = torch.zeros((1, 4, 4, D), device="cuda")
    with pytest.raises(ShapeError):
        c.tree_decode(q)  # fewer positions than drafts
    x = torch.zeros((1, 10, 2, D), device="cuda")
    c.append(x, x)
    c.tree_decode(q)
    for bad in (q.half(), q.cpu(), q[0], torch.zeros((2, 4, 4, D), device="cuda"),
                torch.zeros((1, 4, 3, D), device="cuda"), torch.zeros((1, 4, 0, D), device="cuda")):
        with pytest.raises(ShapeError):
            c.tree_decode(bad)
    with pytest.raises(UnsupportedError):
        c.tree_decode(torch.zeros((1, 65, 4, D), device="cuda"))
    with pytest.raises(ShapeError):
        c.tree_decode(q, torch.zeros((1, 4), dtype=torch.int64))
    p = paged.PagedKv3Cache(1, 4, 2)
    r = p.create_request()
    p.append(0, [r], x[:, :3], x[:, :3])
    with pytest.raises(ShapeError):
        p.tree_decode(0, [r], q)
    assert p.tree_decode(0, [], torch.zeros((0, 4, 4, D), device="cuda")).shape == (0, 4, 4, D)
    c.close()
    p.close()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_splits(kv, dtype):
    """One kv head over 40007 positions: every CTA of the GPU takes a split."""
    g = generator(31)
    n, T, Hq = 40007, 5, 2
    c = kv.Kv3Cache(1, 1, n)
    c.append(rand(g, 1, n, 1, D), rand(g, 1, n, 1, D))
    q = (2 * rand(g, 1, T, Hq, D)).to(dtype)
    mask, bits = rand_mask(g, 1, T)
    k, v = c.get_range(0, n)
    check(c.tree_decode(q, mask)[0], exact(q[0], k[0], v[0], bits[0]), dtype, "R", n)
    c.close()


def test_paged_calls_refuse_a_capture(paged):
    from ferrisres_b200._lib import UnsupportedError
    g = generator(32)
    p = paged.PagedKv3Cache(1, 12, 2)
    r = p.create_request()
    x = rand(g, 1, 70, 2, D)
    p.append(0, [r], x, x)
    f = p.fork_request(r)
    q = rand(g, 2, 4, 4, D)
    want = p.tree_decode(0, [r, f], q)
    idx = torch.arange(40, 60, dtype=torch.int32, device="cuda")
    w = torch.zeros((2, 2, 70), device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for refused in (lambda: p.tree_decode(0, [r, f], q), lambda: p.keep(0, [f], idx),
                        lambda: p.evict_heavy(0, [r, f], w, 40)):
            with pytest.raises(UnsupportedError):
                refused()
    assert torch.equal(p.tree_decode(0, [r, f], q), want)
    p.ctx.check()
    p.close()


def test_captured_and_replayed(kv):
    g = generator(14)
    c = kv.Kv3Cache(2, 2, 600)
    c.append(rand(g, 2, 600, 2, D), rand(g, 2, 600, 2, D))
    q = rand(g, 2, 7, 8, D)
    mask, _ = rand_mask(g, 2, 7)
    ref = c.tree_decode(q, mask)
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.tree_decode(q, mask, out=out)
    # a larger call grows the workspace; the graph keeps its own
    big = torch.zeros((2, 64, 8, D), device="cuda")
    c.tree_decode(big)
    q2 = rand(g, 2, 7, 8, D)
    want = c.tree_decode(q2, mask)
    for src, res in ((q.clone(), ref), (q2, want)):
        q.copy_(src)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, res)
    c.ctx.check()
    c.close()


def test_same_call_same_bits(kv):
    g = generator(15)
    c = kv.Kv3Cache(1, 8, 9000, mode="T", seed=1)
    c.append(rand(g, 1, 9000, 8, D), rand(g, 1, 9000, 8, D))
    q = rand(g, 1, 16, 32, D).bfloat16()
    a = c.tree_decode(q)
    for _ in range(3):
        assert torch.equal(c.tree_decode(q), a)
    c.close()
