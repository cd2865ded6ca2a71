"""Infinite values that a token does see (mmoe_attn_paged): the result does not depend on which tile or partial result holds them."""
import numpy as np
import pytest

import maplemoe as M
from paged_ref import HALF, Batch, Dev, decode, encode

pytestmark = pytest.mark.gpu
INF = float("inf")

SHAPES = {
    "single token": dict(qlens=[1], lens=[400], heads=4, kv=1),
    "single token, window": dict(qlens=[1], lens=[400], heads=4, kv=1, window=395),
    "single token, chunks": dict(qlens=[1, 1], lens=[2500, 600], heads=4, kv=1),
    "single token, many chunks": dict(qlens=[1], lens=[9000], heads=4, kv=1),
    "row tile": dict(qlens=[60], lens=[300], heads=2, kv=1),
    "row tile, window": dict(qlens=[60], lens=[300], heads=2, kv=1, window=270),
    "row tile, runs": dict(qlens=[60], lens=[1300], heads=2, kv=1),
    "row tile, many runs": dict(qlens=[40], lens=[4200], heads=1, kv=1),
    "shared positions, chunks": dict(qlens=[1, 3], lens=[600, 700], heads=4, kv=1, shared=512),
    "shared positions, row tiles": dict(qlens=[40, 40, 41], lens=[2150, 2200, 2100], heads=8, kv=1, shared=2048),
}


@pytest.mark.parametrize("kind,dim", [("f16", 64), ("bf16", 128)])
@pytest.mark.parametrize("name", list(SHAPES))
def test_an_infinite_value_of_small_weight(name, kind, dim):
    """scores are set by hand (a key's first dim is its score): infinite values 25 and 110 below the largest one, whose weights are 0 in
    16 bits, and in 32 bits, in positions that every row of a tile sees and in positions that only some of them see"""
    c = SHAPES[name]
    b = Batch(np.random.default_rng(len(name) + dim), kind=kind, dim=dim, bs=16, **c)
    rng = np.random.default_rng(3)
    k, v, q = np.zeros(b.k.shape), rng.standard_normal(b.v.shape), np.zeros(b.q.shape)
    q[..., 0] = 1.0
    k[..., 0] = 0.25 * rng.integers(-4, 5, k.shape[:-1])
    b.scale = 1.0

    def put(s, p, score, value=None, dims=slice(0, 0)):
        at = b.table[s, p // b.bs], p % b.bs
        k[at][:, 0] = score
        if value is not None:
            v[at][:, dims] = value
    n = len(b.lens)
    for s in range(n):
        end = b.lens[s]
        if s == 0:   # what every sequence sees where positions are shared
            put(0, 33, -25.0, INF, slice(3, 9))
            put(0, 34, -25.0, -INF, slice(20, 22))
            put(0, 8, -25.0, INF, slice(30, 31))
            put(0, 40, 0.0, -INF, slice(50, 51))
            put(0, 41, -25.0, INF, slice(51, 53))
        put(s, end - 2, -25.0, INF, slice(40, 41))
        put(s, end - 5, -25.0, -INF, slice(51, 52))
        put(s, end - 30, 110.0)       # behind them: the weights of everything before it are 0 from here on
    b.k, b.v, b.q = (encode(x, kind) for x in (k, v, q))
    with Dev() as d:
        a = b.upload(d)
        M.check(d.lib.mmoe_attn_paged(a, b.cache), "attention")
        b.check(d, name)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("qlens,lens,shared", [([1], [700], 0), ([2, 90], [300, 400], 0), ([50, 40, 30], [1290, 1240, 1230], 1024)])
@pytest.mark.parametrize("log", [13, 18, 22, 24, 25, 26, 27, 29, 40])
def test_large_scores(log, qlens, lens, shared, kind):
    """a row's scores are all equal, 2^log to 2^(log + 1) of either sign: its result is its values' mean, as near as scores in 32 bits tell,
    and, where they tell nothing (a step of theirs is more than the exponentials' range), between its values"""
    b = Batch(np.random.default_rng(17), kind=kind, heads=8, kv=1, dim=64, qlens=qlens, lens=lens, shared=shared)
    rng = np.random.default_rng(18)
    k, q = np.zeros(b.k.shape), np.zeros(b.q.shape)
    k[..., 0] = 8.0
    size = 1 + rng.integers(0, 128, q.shape[:2]) / 128
    q[..., 0] = size * rng.choice([-1, 1], size.shape)
    b.scale = 2.0 ** (log - 3)
    b.k, b.q = encode(k, kind), encode(q, kind)
    with Dev() as d:
        a = b.upload(d)
        M.check(d.lib.mmoe_attn_paged(a, b.cache), "attention")
        got = decode(d.get(b.p_out, b.out0)[:, 8:8 + 8 * 72].reshape(b.ntok, 8, 72)[..., :64].copy(), kind)
    assert np.isfinite(got).all()
    for s in range(len(lens)):
        v = b.cached(s)[1][:, 0]
        for t in range(b.qstart[s], b.qstart[s + 1]):
            see = v[:b.pos[t] + 1]
            mean, mag, low, high = see.mean(0), np.abs(see).mean(0), see.min(0), see.max(0)
            # a result's rounding and a weight's, 2^-21 for 32-bit sums; a score's product, maximum and difference: three roundings
            e = (3 * 2.0 ** -24 * size[t] * 2.0 ** log)[:, None]
            near = np.abs(got[t] - mean) <= HALF[kind] * np.abs(mean) + (HALF[kind] + 2.0 ** -21 + np.expm1(np.minimum(2 * e, 9))) * mag
            wide = 2 * HALF[kind] * np.abs(see).max(0)
            assert np.where(e < 0.5, near, (got[t] >= low - wide) & (got[t] <= high + wide)).all(), (s, t)


@pytest.mark.parametrize("qlens,lens", [([1], [700]), ([2, 90], [300, 400])])
@pytest.mark.parametrize("log", [22, 23, 24, 25, 26, 27])
def test_large_scores_some_steps_apart(log, qlens, lens):
    """scores as above; those of the later positions lie zero to three of their own steps in 32 bits higher: results stay between the values"""
    b = Batch(np.random.default_rng(27), kind="f16", heads=8, kv=1, dim=64, qlens=qlens, lens=lens)
    rng = np.random.default_rng(28)
    k, q = np.zeros(b.k.shape), np.zeros(b.q.shape)
    k[..., 0] = 8.0
    for s in range(len(lens)):
        for p in range(lens[s] // 3, lens[s]):
            k[b.table[s, p // b.bs], p % b.bs, :, 1] = 2.0 ** -10 * rng.integers(0, 4)
    q[..., 0] = 1 + rng.integers(0, 128, q.shape[:2]) / 128
    q[..., 1] = 2.0 ** -10    # products in steps of 2^-20: the last bit of 8 to 16
    b.scale = 2.0 ** (log - 3)
    b.k, b.q = encode(k, "f16"), encode(q, "f16")
    with Dev() as d:
        a = b.upload(d)
        M.check(d.lib.mmoe_attn_paged(a, b.cache), "attention")
        got = decode(d.get(b.p_out, b.out0)[:, 8:8 + 8 * 72].reshape(b.ntok, 8, 72)[..., :64].copy(), "f16")
    assert np.isfinite(got).all()
    for s in range(len(lens)):
        v = b.cached(s)[1][:, 0]
        for t in range(b.qstart[s], b.qstart[s + 1]):
            see = v[:b.pos[t] + 1]
            wide = 2 * HALF["f16"] * np.abs(see).max(0)
            assert ((got[t] >= see.min(0) - wide) & (got[t] <= see.max(0) + wide)).all(), (s, t)


@pytest.mark.parametrize("scale,slope,cap", [(1e-20, 1e8, 0.0), (1e-20, 1e8, 50.0), (1e-20, -1e8, 0.0), (1e20, 0.5, 0.0), (1e20, 0.5, 4.0), (1e20, 1e8, 0.0)])
@pytest.mark.parametrize("qlens,lens", [([1], [700]), ([50, 2], [300, 90])])
def test_scales_and_slopes_at_their_limits(scale, slope, cap, qlens, lens):
    b = Batch(np.random.default_rng(9), kind="bf16", heads=4, kv=1, dim=64, qlens=qlens, lens=lens, alibi=True, cap=cap)
    b.slopes = (b.slopes * np.float32(slope)).astype(np.float32)
    b.scale = scale
    if scale > 1:
        b.q = encode(np.random.default_rng(10).standard_normal(b.q.shape) / scale, "bf16")
    with Dev() as d:
        a = b.upload(d)
        M.check(d.lib.mmoe_attn_paged(a, b.cache), "attention")
        b.check(d, f"scale {scale} slope {slope} cap {cap}")
