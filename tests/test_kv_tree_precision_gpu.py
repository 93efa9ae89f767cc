"""Where the tree decode's 16-bit operands could lose bits or overflow: results against attention in 64
bits over the stored values (``exact`` and its X, V are those of test_kv_tree_gpu).

Bounds, each an upper limit of the roundings that the formula needs:
  scores: K vectors here are a level plus little noise, so that a score is level * sum(q) (fp32: qsum, the
    factor and the product, 4 roundings of 2^-24 and the sum of 128 terms, 2^-22 together) plus a small
    product of codes: below 2^-20 * X.  p is off by twice that, X <= 40 in these tests where nothing else
    is said: 2^-19 * 40 / 4 in the 2-norm (rounding errors of both signs) = 2e-5 at most; where X <= 20, 1e-5.
  weights: fp16 hi + lo of p (max - min)/7: relative 2^-22, absolute 2^-25 of a largest of at least 2^5.
  bf16 output: half a step, 2^(floor(log2 |out|) - 8), plus the fp32 error before it.
"""
import pytest
import torch

from test_kv_tree_gpu import (D, causal_bits, check, exact, generator, kv, paged, rand,  # noqa: F401
                              rand_mask)

pytestmark = pytest.mark.gpu


def ring(kv, k, v, mode="R", seed=3):
    c = kv.Kv3Cache(k.shape[0], k.shape[2], k.shape[1], mode=mode, seed=seed)
    c.append(k, v)
    return c


def near(got, ref, rel):
    out = ref[0]
    assert bool(torch.isfinite(got.float()).all())
    err = float((got.double() - out).norm() / out.norm())
    assert err <= rel, err


def half_step(x):
    """Half a step of bf16 at |x| (x in 64 bits)."""
    return torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(1e-30))) - 8)


# ------------------------------------------------------------ bf16 queries --
@pytest.mark.parametrize("n", [64, 66, 200, 1500])
def test_bf16_output_is_rounded_once(kv, n):
    """bf16 queries: the output is the fp32 result rounded once.  Small scores (X about 1.3) make the fp32
    error small: 2 * 3 X 2^-20 of the scores, 2^-18 and 2^-21 of the exponentials and weights, sums of
    (n / 32 + 16) 2^-24 of 3 V.  An output may differ from the rounded exact result only where that lies
    within the error of a rounding border, which of m outputs happens to sum(error / half step) at most."""
    g = generator(n)
    T, Hq, H = 64, 8, 2
    c = ring(kv, rand(g, 1, n, H, D), rand(g, 1, n, H, D))
    q = (0.05 * rand(g, 1, T, Hq, D)).bfloat16()
    bits = torch.eye(T, dtype=torch.bool, device="cuda")  # a draft sees the prefix and itself
    mask = torch.ones(T, dtype=torch.int64, device="cuda") << torch.arange(T, device="cuda")
    got = c.tree_decode(q, mask)[0].double()
    k, v = c.get_range(0, n)
    out, X, V = exact(q[0], k[0], v[0], bits)
    tol = V * (6 * X * 2.0 ** -20 + 2.0 ** -18 + 2.0 ** -21 + 3 * (n / 32 + 16) * 2.0 ** -24)
    half = half_step(out.abs() + tol)
    assert bool(((got - out).abs() <= half + tol).all())
    differ = int((got != out.float().bfloat16().double()).sum())
    expected = float((tol / half_step(out)).clamp_max(1).sum())
    assert differ <= expected + 6 * expected ** 0.5, (differ, expected, got.numel())
    c.close()


@pytest.mark.parametrize("n,T,Hq,H", [(5, 5, 8, 2), (64, 64, 8, 8), (128, 21, 10, 2), (100, 64, 16, 1)])
def test_bf16_queries_in_mode_t(kv, n, T, Hq, H):
    """The rotated query is no bf16 value: it is taken with the bits of an fp32 one.  The same q as fp32
    gives the same result before the one rounding (one tile of positions: one split either way)."""
    g = generator(n + T)
    c = ring(kv, rand(g, 2, n, H, D), rand(g, 2, n, H, D), mode="T")
    q = (2 * rand(g, 2, T, Hq, D)).bfloat16()
    assert torch.equal(c.tree_decode(q), c.tree_decode(q.float()).bfloat16())
    c.close()


# ------------------------------------------------- references of the softmax --
def levels(g, n, H, at):
    """K whose score is level * sum(q): at [n] in units of log2 for a q of ones, and q rows near ones."""
    unit = 1.4426950408889634 * D ** 0.5  # log2 of a score per unit of level, sum(q) = 128
    return (at / unit)[None, :, None, None] + 0.01 * rand(g, 1, n, H, D)


def test_weights_that_fall_by_2_to_26_within_a_tile(kv):
    """One record grows the reference's headroom, the next passes it by 2^18: what the records before hold
    in 16 bits is scaled by 2^-26, and counts for 64 * 2^-18 of the result."""
    g = generator(41)
    n, T, H, Hq = 128, 1, 1, 80  # above 64 rows a row takes all records of a tile
    at = torch.zeros(n, device="cuda")
    at[32:96] = 7.3
    at[96:] = -10.0
    at[100] = 7.3 + 18.9
    k = levels(g, n, H, at)
    v = rand(g, 1, n, H, D)
    v[:, 32:96] = rand(g, 1, 1, H, D)
    c = ring(kv, k, v)
    q = 1 + 0.02 * rand(g, 1, T, Hq, D)
    kk, vv = c.get_range(0, n)
    ref = exact(q[0], kk[0], vv[0], causal_bits(1, T)[0])
    near(c.tree_decode(q)[0], ref, 1e-5)
    c.close()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("power", [12, 17, 22, 27, 40])
def test_values_of_one_position_far_above_the_others(kv, power, dtype):
    """A position whose values are 2^power times its neighbours' and whose weight is 2^-60: it takes no
    bits from theirs."""
    g = generator(power)
    n, T, H, Hq = 300, 2, 2, 8
    at = torch.zeros(n, device="cuda")
    at[32:] = 8.0
    at[70] = at[150] = -56.0
    k, v = levels(g, n, H, at), rand(g, 1, n, H, D)
    for i in (70, 150):
        v[:, i] *= 2.0 ** power
    c = ring(kv, k, v)
    q = (1 + 0.02 * rand(g, 1, T, Hq, D)).to(dtype)
    kk, vv = c.get_range(0, n)
    ref = exact(q[0], kk[0], vv[0], causal_bits(1, T)[0])
    near(c.tree_decode(q)[0], ref, 2e-5 if dtype == torch.float32 else 0.6 * 2.0 ** -8)
    c.close()


@pytest.mark.parametrize("size", [0.0, 1e-4, 1e-2])
@pytest.mark.parametrize("share", [6, 10, 14, 20])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_sink(kv, dtype, share, size):
    """Position 0 takes all but 2^-share of the weight and has values of `size`: the others' weights keep
    their bits."""
    g = generator(share)
    n, T, H, Hq = 512, 1, 2, 8
    at = torch.zeros(n, device="cuda")
    at[0] = share + 9
    k, v = levels(g, n, H, at), rand(g, 1, n, H, D)
    v[:, 0] *= size
    c = ring(kv, k, v)
    q = (1 + 0.02 * rand(g, 1, T, Hq, D)).to(dtype)
    kk, vv = c.get_range(0, n)
    ref = exact(q[0], kk[0], vv[0], causal_bits(1, T)[0])
    near(c.tree_decode(q)[0], ref, 2e-5 if dtype == torch.float32 else 0.6 * 2.0 ** -8)
    c.close()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 31, 1024])
@pytest.mark.parametrize("value", [3.0, 1e9, 1e11, -1e20, 1e30, 1e38, 1e-20])
def test_constant_values_of_any_size(kv, value, n, dtype):
    """V vectors without a range (step 0): the result is the value, for all sizes that have one."""
    g = generator(n)
    k = rand(g, 1, n, 2, D)
    c = ring(kv, k, torch.full_like(k, value))
    q = rand(g, 1, 1, 4, D).to(dtype)
    got = c.tree_decode(q).double()
    kk, vv = c.get_range(0, n)
    want = vv.double().mean()
    assert float((got - want).abs().max()) <= (1e-5 if dtype == torch.float32 else 2.0 ** -8) * abs(float(want))
    c.close()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [1e-25, 1e-20, 1e30, 1e34, 1e37])
def test_value_ranges_up_to_the_largest(kv, size, dtype):
    """V of sizes up to the largest whose range is finite, with weights that spread over 2^20."""
    g = generator(43)
    n, T, H, Hq = 300, 2, 1, 4
    at = -20 * torch.rand((n,), generator=g, device="cuda")
    k, v = levels(g, n, H, at), rand(g, 1, n, H, D) * size
    c = ring(kv, k, v)
    q = (1 + 0.02 * rand(g, 1, T, Hq, D)).to(dtype)
    kk, vv = c.get_range(0, n)
    ref = exact(q[0], kk[0], vv[0], causal_bits(1, T)[0])
    near(c.tree_decode(q)[0], ref, 2e-5 if dtype == torch.float32 else 0.6 * 2.0 ** -8)
    c.close()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("flip", [False, True])
@pytest.mark.parametrize("far", [64, 700, 3000])
def test_constant_values_beside_very_large_ones(kv, far, flip, dtype):
    """Half of the positions with constant values, half with a range of 1e34, equal scores: references
    that lie 2^190 apart meet within a tile, between groups and between splits."""
    g = generator(far)
    n = 2 * far
    k, v = levels(g, n, 1, torch.zeros(n, device="cuda")), torch.ones((1, n, 1, D), device="cuda")
    v[:, :far] = rand(g, 1, far, 1, D) * 1e34
    if flip:
        v = v.flip(1).contiguous()
    c = ring(kv, k, v)
    q = (1 + 0.02 * rand(g, 1, 1, 4, D)).to(dtype)
    kk, vv = c.get_range(0, n)
    ref = exact(q[0], kk[0], vv[0], causal_bits(1, 1)[0])
    near(c.tree_decode(q)[0], ref, 2e-5 if dtype == torch.float32 else 0.6 * 2.0 ** -8)
    c.close()


@pytest.mark.parametrize("kind", ["rise", "fall", "steps", "huge", "values", "constant", "jumps", "spikes"])
def test_references_that_move_fp32(kv, kind):
    """fp32 queries: scores and value ranges that move by a little and by a lot, between tiles and between
    the records of one.  p is off by twice 3 X 2^-20 at most (the scores' bound); terms add up to 2 V."""
    g = generator(22)
    n, T, Hq, H = 2500, 6, 8, 2
    k, v = rand(g, 1, n, H, D), rand(g, 1, n, H, D)
    q = 2 * rand(g, 1, T, Hq, D)
    at = torch.arange(n, device="cuda")[None, :, None, None]
    along = torch.nn.functional.normalize(q.mean((1, 2)), dim=-1)  # moves every row's score
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
    elif kind == "constant":
        v[:, ::2] = 0.5
        v[:, 1200:1600] = 0.0
        k[:, 700] = 1.0
    elif kind == "jumps":  # score and range change by up to 2^30 between records of a tile
        k = k + along * (at // 32 * 7 % 5)
        v = v * torch.exp2((at // 32 * 17 % 30).float())
    else:
        v[:, 5::97] *= 2.0 ** 20
        k[:, 5::97] -= along * 8
    c = ring(kv, k, v)
    got = c.tree_decode(q)[0].double()
    c.ctx.check()
    kk, vv = c.get_range(0, n)
    out, X, V = exact(q[0], kk[0], vv[0], causal_bits(1, T)[0])
    tol = V * (6 * X * 2.0 ** -20 + 2.0 ** -18 + 2.0 ** -21 + 3 * (n / 32 + 16) * 2.0 ** -24)
    assert bool(((got - out).abs() <= tol).all())
    c.close()


@pytest.mark.parametrize("mode", ["R", "T"])
@pytest.mark.parametrize("case", [(1, 128 + 1, 1, 1, 1), (1, 256 + 3, 2, 8, 2), (2, 385, 1, 16, 2), (1, 1100, 4, 32, 8),
                                  (1, 2100, 64, 2, 1), (2, 1500, 64, 4, 1), (1, 3000, 33, 20, 4), (3, 900, 64, 15, 3),
                                  (1, 20000, 8, 8, 2), (8, 640, 17, 8, 8)])
def test_whole_prefix_tiles_fp32(kv, case, mode):
    """fp32 queries, the cases that test_kv_tree_gpu has for bf16 ones: one and many tiles, few and many rows,
    heads and channels of unequal spread.  Bounds: test_kv_tree_gpu."""
    B, n, T, Hq, H = case
    g = generator(n + T)
    spread = 0.2 + 2 * torch.rand((H, D), generator=g, device="cuda")
    c = ring(kv, rand(g, B, n, H, D) * spread, rand(g, B, n, H, D) * spread, mode=mode)
    q = 2 * rand(g, B, T, Hq, D)
    mask, bits = rand_mask(g, B, T)
    out = c.tree_decode(q, mask)
    c.ctx.check()
    k, v = c.get_range(0, n)
    for b in range(B):
        check(out[b], exact(q[b], k[b], v[b], bits[b]), torch.float32, mode, n)
    c.close()
