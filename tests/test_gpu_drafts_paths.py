"""Drafted tokens on the card (include/maplemoe.h, Part 3), by how a call is divided: whole row tiles and pieces, few of them and more than there is room
for, joins of either kind, batches past 64 sequences; infinite values, wherever they lie; long lists of kept positions."""
import numpy as np
import pytest

import maplemoe as M
from draft_ref import TreeBatch, compact, paths, tree
from paged_ref import Dev, encode
from test_gpu_pages import Layers, table_of

pytestmark = pytest.mark.gpu
INF = float("inf")


def drafts(rng, sizes, back):
    return [paths(tree(rng, n, back)) for n in sizes]


MANY = {  # nodes of sequence s, cached positions of sequence s, sequences, options
    "70 sequences, few long": (lambda s: 1 + s % 3, lambda s: 6000 if s in (3, 65) else 20 * s, 70, dict(heads=4, kv=1)),
    "300 sequences": (lambda s: s % 3, lambda s: 300 + 7 * (s % 90), 300, dict(heads=2, kv=2, dim=64, kind="bf16")),
    "70 sequences, shared": (lambda s: 1 + s % 9, lambda s: 512 + 3 * s, 70, dict(heads=8, kv=2, shared=512)),
    "300 sequences, shared": (lambda s: 1 + s % 2, lambda s: 64 + s % 50, 300, dict(heads=4, kv=1, dim=64, shared=64, kind="bf16")),
    "more row tiles than room": (lambda s: 10, lambda s: 30 + 11 * (s % 80), 80, dict(heads=64, kv=1, dim=64)),
    "more row tiles than room, 60 sequences": (lambda s: 1 + s % 3, lambda s: 15 * s, 60, dict(heads=8, kv=8, kind="bf16")),
    "more key/value heads than pieces": (lambda s: 2, lambda s: 400 + 100 * s, 3, dict(heads=520, kv=520, dim=64)),
    "whole, window": (lambda s: 1 + s % 4, lambda s: 9 * s, 200, dict(heads=2, kv=1, window=100)),
    "whole, 64 sequences": (lambda s: 2 + s % 3, lambda s: 5 * s, 64, dict(heads=8, kv=4, dim=64, kind="bf16", alibi=True)),
    "pieces joined by rows": (lambda s: 3 + s, lambda s: 3000 + 100 * s, 8, dict(heads=8, kv=4)),
    "pieces joined by rows, heads of 64": (lambda s: 3 + s, lambda s: 3000 - 300 * s, 9, dict(heads=8, kv=4, dim=64, kind="bf16")),
    "900 sequences, most without tokens": (lambda s: 7 if s % 30 == 11 else 0, lambda s: 40 * s if s % 30 == 11 else 9, 900, dict(heads=8, kv=2, pad=500, max_q=64)),
    "900 sequences, most without tokens, shared": (lambda s: 2 if s % 100 == 50 else 0, lambda s: 128 + s, 900, dict(heads=4, kv=2, shared=128, dim=64, max_q=20)),
    "more pieces than workgroups": (lambda s: 1 + s % 2, lambda s: 10 + s % 60, 700, dict(heads=4, kv=4, dim=64, kind="bf16")),
    "more pieces than workgroups, cut": (lambda s: 1, lambda s: 700 + s, 160, dict(heads=6, kv=6, dim=64, alibi=True)),
    "one long, the others none": (lambda s: 2 if s == 40 else 0, lambda s: 8000 if s == 40 else 50, 64, dict(heads=4, kv=2)),
}


@pytest.mark.parametrize("name", list(MANY))
def test_division(name):
    nodes, ctx, n, kw = MANY[name]
    print(f"\n  {name}", flush=True)
    rng = np.random.default_rng(len(name))
    sizes = [nodes(s) for s in range(n)]
    b = TreeBatch(rng, drafts(rng, sizes, 3), lens=[ctx(s) + x for s, x in enumerate(sizes)], **kw)
    with Dev() as d:
        b.run(d, name)


SHAPES = {
    "one draft": ([4], [400], dict(heads=4, kv=1)),
    "one draft, window": ([4], [400], dict(heads=4, kv=1, window=392)),
    "one draft, many pieces": ([3], [9000], dict(heads=4, kv=1)),
    "row tile": ([60], [300], dict(heads=2, kv=1)),
    "row tiles, pieces": ([60, 50], [1300, 4200], dict(heads=8, kv=1)),
    "joined by rows": ([3, 5, 4, 6, 7, 3, 9, 8], [2500, 600, 700, 3000, 500, 900, 1200, 700], dict(heads=8, kv=4)),
    "shared positions": ([1, 3], [600, 700], dict(heads=4, kv=1, shared=512)),
    "shared positions, row tiles": ([40, 40, 41], [2150, 2200, 2100], dict(heads=8, kv=1, shared=2048)),
    "whole": ([2] * 200, [120 + s % 9 for s in range(200)], dict(heads=1, kv=1)),
}


@pytest.mark.parametrize("kind,dim", [("f16", 64), ("bf16", 128)])
@pytest.mark.parametrize("name", list(SHAPES))
def test_an_infinite_value_of_small_weight(name, kind, dim):
    """scores are set by hand (a key's first dim is its score): infinite values 25 and 110 below the largest one, whose weights are 0 in 16 bits, and
    in 32 bits; cached ones, and drafted ones that only those who follow them see"""
    sizes, lens, kw = SHAPES[name]
    rng = np.random.default_rng(3)
    b = TreeBatch(np.random.default_rng(len(name) + dim), drafts(rng, sizes, 3), lens=lens, kind=kind, dim=dim, bs=16, **kw)
    k, v, q = np.zeros(b.k.shape), rng.standard_normal(b.v.shape), np.zeros(b.q.shape)
    q[..., 0] = 1.0
    k[..., 0] = 0.25 * rng.integers(-4, 5, k.shape[:-1])
    b.scale = 1.0

    def put(s, p, score, value=None, dims=slice(0, 0)):
        at = b.table[s, p // b.bs], p % b.bs
        k[at][:, 0] = score
        if value is not None:
            v[at][:, dims] = value
    for s in range(len(lens)):
        end, ctx = lens[s], lens[s] - sizes[s]
        if s == 0:   # what every sequence sees where positions are shared
            put(0, 33, -25.0, INF, slice(3, 9))
            put(0, 34, -25.0, -INF, slice(20, 22))
            put(0, 8, -25.0, INF, slice(30, 31))
            put(0, 40, 0.0, -INF, slice(50, 51))
            put(0, 41, -25.0, INF, slice(51, 53))
        put(s, ctx + sizes[s] // 2, -25.0, INF, slice(40, 41))
        put(s, ctx + sizes[s] - 1, -25.0, -INF, slice(42, 43))
        put(s, ctx - 5, -25.0, -INF, slice(51, 52))
        put(s, ctx - 30, 110.0)       # behind them: the weights of everything before it are 0 from here on
    b.k, b.v, b.q = (encode(x, kind) for x in (k, v, q))
    with Dev() as d:
        b.run(d, name)


# ---------------------------------------------------------------------------------------------------- kept positions, long lists
@pytest.mark.parametrize("kw,n,length,part", [
    (dict(layers=128, kv=1, dim=64, bs=32), 4, 700, 0.4),               # workgroups of 256
    (dict(layers=24, kv=8, dim=64, token_major=True), 3, 500, 0.5),
    (dict(layers=20, kv=2, dim=8, gap=0), 20, 250, 0.6),                # one piece a head: pieces in twos
    (dict(layers=1, kv=1, dim=64), 1, 9000, 0.9),                       # of 1024, several steps
    (dict(layers=3, kv=4, dim=128, kind="f32"), 2, 2500, 0.5),
    (dict(layers=2, kv=3, dim=72), 5, 900, 0.3)])
def test_compact_long_lists(kw, n, length, part):
    print(f"\n  {kw} {n} sequences of {length}", flush=True)
    rng = np.random.default_rng(n * 37 + length)
    bs = kw.get("bs", 16)
    width = -(-length // bs)
    with Dev() as d:
        c = Layers(d, rng, nblocks=n * width, **kw)
        table = table_of(rng, n, width, c.nblocks)
        lists = [np.sort(rng.permutation(length)[:max(1, int(length * part))]) for _ in range(n)]
        count = np.array([len(x) for x in lists], np.int32)
        first, kept = (np.cumsum(count) - count).astype(np.int32), np.concatenate(lists).astype(np.int32)
        a = M.KvCompact(table=d.put(table), first=d.put(first), count=d.put(count), kept=d.put(kept), nseq=n, width=width, nkept=len(kept))
        M.check(d.lib.mmoe_kv_compact(a, c.caches, c.n), "mmoe_kv_compact")
        c.check(lambda x: compact(x, table, first, count, kept, len(kept), bs), str(kw))
