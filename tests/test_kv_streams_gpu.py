"""Cache calls on a stream of their own, while what they read is still being written on the current
one, and temporaries that the allocator could hand out again: results as on one stream."""
import pytest
import torch

pytestmark = pytest.mark.gpu

D = 128


def late(make):
    """Tensors whose values arrive on the current stream only after some 20 ms of waiting there."""
    values = make()
    out = [torch.zeros_like(v) for v in values]
    torch.cuda.synchronize()
    torch.cuda._sleep(40_000_000)
    for o, v in zip(out, values):
        o.copy_(v)
    return out


def wide(t):
    """The same values as every second position of a larger tensor (a call has to lay them out)."""
    w = t.new_zeros((t.shape[0], 2 * t.shape[1], *t.shape[2:]))
    w[:, ::2] = t
    return w


def reuse():
    """Takes what the allocator has free on the current stream and overwrites it."""
    junk = [torch.full((n,), -1, dtype=torch.int32, device="cuda") for n in (16, 256, 4096, 1 << 16, 1 << 18)]
    return junk


def stored(c, *where):
    return [t.clone() for t in c.export_range(*where)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ring(dtype):
    from ferrisres_b200 import kv
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    n, H = 200, 2
    x = [torch.randn((2, n, H, D), generator=g, device="cuda").to(dtype) for _ in range(2)]
    q = torch.randn((2, 4, D), generator=g, device="cuda")
    a = kv.Kv3Cache(2, H, 512)
    a.append(*x)
    packed = stored(a, 0, n)
    a.append_packed(*packed)
    want, full = a.flash_decode(q), stored(a, 0, 2 * n)
    kept = torch.arange(50, 150, dtype=torch.int32, device="cuda")
    a.keep(kept)
    want_kept = stored(a, 0, 100)

    side = torch.cuda.Stream()
    c = kv.Kv3Cache(2, H, 512)
    k, v = late(lambda: [wide(t) for t in x])
    c.append(k[:, ::2], v[:, ::2], stream=side)
    junk = reuse()
    t = late(lambda: [wide(t) for t in packed])
    c.append_packed(*[s[:, ::2] for s in t], stream=side)
    junk += reuse()
    got = c.export_range(0, 2 * n, stream=side)
    (qq,) = late(lambda: [q])
    out = c.flash_decode(qq, stream=side)
    values = c.get_range(0, 2 * n, stream=side)
    (ii,) = late(lambda: [kept.long()])
    c.keep(ii, stream=side)
    junk += reuse()
    after = c.export_range(0, 100, stream=side)
    side.synchronize()
    assert all(torch.equal(s, t) for s, t in zip(got, full))
    assert torch.equal(out, want)
    assert all(torch.equal(s, t) for s, t in zip(after, want_kept))
    assert all(bool(torch.isfinite(t).all()) for t in values)
    c.ctx.check()
    a.close()
    c.close()


def test_paged():
    from ferrisres_b200 import paged
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    n, H = 100, 2
    x = [torch.randn((2, n, H, D), generator=g, device="cuda") for _ in range(2)]
    q = torch.randn((2, 4, D), generator=g, device="cuda")
    w0 = torch.rand((2, H, 2 * n), generator=g, device="cuda")

    def run(stream, given):
        c = paged.PagedKv3Cache(1, 40, H)
        r = c.create_request()
        (k, v), packed, qq, w = given()
        c.append(0, [r], k[:1], v[:1], stream=stream)
        f = c.fork_request(r)
        c.append(0, [f, r], k[:, ::2], v[:, ::2], stream=stream)  # copies the shared page first
        junk = reuse()
        c.append_packed(0, [r, f], *[t[:, ::2] for t in packed], stream=stream)
        junk += reuse()
        m = c.seq_len(r)
        res = [*c.export_range(0, [r, f], 0, m, stream=stream), *c.get_range(0, [f], 3, m, stream=stream)]
        res.append(c.flash_decode(0, [f, r], qq, stream=stream, weights=w))
        res.append(c.flash_decode(0, [r, f], qq, stream=stream))
        res += [w, *c.evict_heavy(0, [r, f], w, 77, 10, stream=stream)]
        res += c.export_range(0, [f, r], 0, 77, stream=stream)
        junk += reuse()
        torch.cuda.synchronize()
        c.ctx.check()
        res = [t.clone() for t in res]
        c.close()
        return res

    source = paged.PagedKv3Cache(1, 40, H)
    rr = [source.create_request() for _ in range(2)]
    source.append(0, rr, *x)
    packed = stored(source, 0, rr, 0, 40)
    source.close()
    m = n + 50 + 40
    plain = lambda: (x, [wide(t) for t in packed], q, w0[:, :, :m].clone())  # noqa: E731

    def slow():
        t = late(lambda: [*x, *[wide(p) for p in packed], q, w0[:, :, :m].clone()])
        return t[:2], t[2:6], t[6], t[7]

    for a, b in zip(run(None, plain), run(torch.cuda.Stream(), slow)):
        assert torch.equal(a, b)
