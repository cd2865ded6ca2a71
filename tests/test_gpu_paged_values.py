"""Infinite values that a token does see (mmoe_attn_paged): the result does not depend on which tile or partial result holds them."""
import numpy as np
import pytest

import maplemoe as M
from paged_ref import Batch, Dev, encode

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
