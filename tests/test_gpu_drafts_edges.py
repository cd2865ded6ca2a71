"""Drafted tokens on the card (include/maplemoe.h, Part 3), at the ends of what the header allows."""
import numpy as np
import pytest

import maplemoe as M
from draft_ref import TreeBatch, tree, tree_plan
from paged_ref import HALF, Dev, attend, decode, encode
from test_gpu_drafts import drafts, run_tree_plan

pytestmark = pytest.mark.gpu
LEAST = -2 ** 31


@pytest.mark.parametrize("sizes,words", [([130], 3), ([512, 200, 65], 8), ([256] * 3, 4)])
@pytest.mark.parametrize("none", [LEAST, LEAST + 1, LEAST + 63, LEAST + 64, LEAST + 447, LEAST + 448, -64, -65])
def test_parents_near_the_smallest_number(sizes, words, none):
    """nodes of every word that follow nobody, whatever negative number says so: the first one of a word, one in its middle, the last one"""
    print(f"\n  {sizes} parent={none}", flush=True)
    rng = np.random.default_rng(len(sizes) + words)
    qstart = np.concatenate([[0], np.cumsum(sizes)])
    parent = np.concatenate([tree(rng, n, 9) for n in sizes]).astype(np.int64)
    for t0, n in zip(qstart, sizes):
        for i in (0, 3, 64, 70, 127, 128, 191, 192, 255, 448, 449, 511):
            if i < n:
                parent[t0 + i] = none
    length = np.array(sizes) + rng.integers(0, 1 << 29, len(sizes))
    got, want = run_tree_plan(qstart, length, parent, words, len(parent)), tree_plan(qstart, length, parent, words, len(parent))
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


KEPT = {  # nodes of sequence s, cached positions of sequence s, sequences, options
    "cut and shared, few of 400 with tokens": (lambda s: 20 if s % 40 == 7 else 0, lambda s: 3000 - 5 * s if s % 40 == 7 else 70, 400, dict(heads=8, kv=2, shared=64, pad=40)),
    "row tiles, cut and shared": (lambda s: 30 - 3 * s, lambda s: 130 + 400 * s, 6, dict(heads=16, kv=1, shared=128, kind="bf16")),
    "row tiles, cut and shared, 66 sequences": (lambda s: 27 if s in (3, 64) else s % 2, lambda s: 2500 if s == 64 else 70, 66, dict(heads=24, kv=2, dim=64, shared=64)),
    "one row short of a wave, one over": (lambda s: (7, 8, 9, 31, 32, 33)[s % 6], lambda s: 300 * (s % 7), 12, dict(heads=4, kv=1)),
    "one row short of a wave, one over, shared": (lambda s: (31, 32, 33, 1, 64, 63)[s], lambda s: 256 + 300 * s, 6, dict(heads=2, kv=2, dim=64, shared=256, kind="bf16")),
    "uncut row tiles, shared": (lambda s: 1 + s % 5, lambda s: 64 + s % 50, 300, dict(heads=12, kv=4, shared=64)),
    "fewer tokens than sequences": (lambda s: int(s == 2000), lambda s: 900 if s == 2000 else 3, 4096, dict(heads=4, kv=1, kind="bf16")),
}


@pytest.mark.parametrize("name", list(KEPT))
def test_results_kept(name):
    """partial results lie wave by wave: row tiles of several waves beside ones of a part of one, with shared positions before them; nothing behind the workspace"""
    nodes, ctx, n, kw = KEPT[name]
    print(f"\n  {name}", flush=True)
    rng = np.random.default_rng(len(name))
    sizes = [nodes(s) for s in range(n)]
    b = TreeBatch(rng, drafts(rng, sizes, 4), lens=[ctx(s) + x for s, x in enumerate(sizes)], **kw)
    with Dev() as d:
        b.run(d, name)


HIDDEN = {  # nodes, lengths, positions whose score is -inf, the one of them that holds infinities, options
    "whole": ([2] * 200, [300] * 200, (0, 250), 70, dict(heads=1, kv=1)),
    "one draft, a piece and more": ([20], [6000], (0, 3000), 1500, dict(heads=4, kv=1)),
    "one draft, the middle": ([20], [6000], (2000, 5000), 3333, dict(heads=8, kv=2)),
    "joined by rows": ([30] * 10, [2500] * 10, (300, 2400), 1700, dict(heads=16, kv=4)),
    "the shared positions": ([5, 30], [2600, 3000], (0, 2048), 999, dict(heads=4, kv=1, shared=2048)),
    "many sequences": ([3] * 70, [3000] * 70, (0, 2900), 1, dict(heads=4, kv=2)),
}


@pytest.mark.parametrize("kind,dim", [("f16", 64), ("bf16", 128)])
@pytest.mark.parametrize("name", list(HIDDEN))
def test_infinite_values_where_every_score_is_minus_infinity(name, kind, dim):
    """a part of the positions as long as a piece or longer has scores of -inf, and an infinite value among them reaches every token that sees it, however
    the call is divided; the other dims are what they are without it, but for the order of their sums: within the bound of either"""
    nodes, lens, (p0, p1), at, kw = HIDDEN[name]
    print(f"\n  {name} {kind}", flush=True)
    rng = np.random.default_rng(len(name) + dim)
    b = TreeBatch(rng, drafts(rng, nodes, 3), lens=lens, kind=kind, dim=dim, **kw)
    b.scale = 1.0
    k, q = 0.3 * decode(b.k, kind), decode(b.q, kind)
    q[..., 0], k[..., 0] = 1.0, 0.0
    for s in range(len(lens)):
        p = np.arange(p0, p1)
        k[b.table[s, p // b.bs], p % b.bs] = 0.0
        k[b.table[s, p // b.bs], p % b.bs, :, 0] = -np.inf
    b.k, b.q = encode(k, kind), encode(q, kind)
    with Dev() as d:
        b.run(d, "finite values")
        want, _, off, _ = b.expect()
        v = decode(b.v, kind)
        for s in range(len(lens)):
            v[b.table[s, at // b.bs], at % b.bs, :, 5] = np.inf
            v[b.table[s, at // b.bs], at % b.bs, :, 6] = -np.inf
            v[b.table[s, at // b.bs], at % b.bs, :, 7] = np.nan
        b.v = encode(v, kind)
        a = b.upload(d)
        M.check(d.lib.mmoe_attn_tree(a, b.cache, b.p_bits, b.words), "attention")
        out = d.get(b.p_out, b.out0)
    n, h = b.ntok, b.heads
    got = decode(out[:, 8:8 + h * (dim + 8)].reshape(n, h, dim + 8)[..., :dim].copy(), kind)
    assert (got[..., 5] == np.inf).all() and (got[..., 6] == -np.inf).all() and np.isnan(got[..., 7]).all()
    rest = [i for i in range(dim) if i not in (5, 6, 7)]
    bad = np.abs(got - want)[..., rest] > off[..., rest]
    assert not bad.any(), np.argwhere(bad)[:5]


# ---------------------------------------------------------------------------------------------------- windows that count along the path
class AlongThePath(TreeBatch):
    """with MMOE_TREE_WINDOW: a token sees itself and the `window` tokens of its path before it, cached or drafted"""

    def expect(self):
        out = np.zeros((self.ntok, self.heads, self.dim))
        lse, off, loff = np.zeros((self.ntok, self.heads)), np.zeros(out.shape), np.zeros((self.ntok, self.heads))
        q = decode(self.q, self.kind)
        for s, rows in enumerate(self.rows):
            k, v = self.cached(s)
            ctx = self.lens[s] - len(rows)
            b = self.table[s][np.arange(self.lens[s]) // self.bs]
            there = (b >= 0) & (b < self.nblocks) & (np.arange(self.lens[s]) < self.max_len)
            for i, row in enumerate(rows):
                t = self.qstart[s] + i
                way = np.array(list(range(ctx)) + [ctx + j for j in range(i) if row[j]] + [ctx + i])
                pos = len(way) - 1
                see = there[way] & (np.arange(len(way)) >= pos - self.window)
                see[:ctx] &= np.arange(ctx) >= (0 if self.lo is None else int(self.lo[t]))
                see[-1] &= bool(row[i])
                with np.errstate(all="ignore"):
                    o, l, e, f = attend(q[t:t + 1], k[way], v[way], np.array([pos]), see[None], self.scale, self.cap, self.slopes, HALF[self.kind])
                out[t], lse[t], off[t], loff[t] = o[0], l[0], e[0], f[0]
        return out, lse, off, loff

    def run(self, d, note=""):
        a = self.upload(d)
        words = self.words | M.TREE_WINDOW
        assert d.lib.mmoe_attn_tree_ws(a, self.cache, self.p_bits, words) == a.ws_bytes
        M.check(d.lib.mmoe_attn_tree(a, self.cache, self.p_bits, words), "mmoe_attn_tree")
        return self.check(d, note)


ALONG = [  # nodes, cached positions, back, options
    ([64, 30, 5], [100, 200, 900], 1, dict(heads=2, kv=1, window=7, kind="bf16")),
    ([64, 30, 5], [100, 200, 900], 2, dict(heads=4, kv=2, window=1)),
    ([64, 64], [100, 200], 1, dict(heads=2, kv=1, window=32)),
    ([61, 20], [70, 190], 2, dict(heads=12, kv=12, dim=64, alibi=True, cap=15.0, window=10)),
    ([130, 140], [600, 128], 1, dict(heads=2, kv=1, window=90, alibi=True, words=3, kind="bf16")),
    ([512, 300], [100, 7], 1, dict(heads=1, kv=1, dim=64, words=8, window=64)),
    ([512], [0], 2, dict(heads=2, kv=1, words=8, window=130, kind="bf16")),
    ([61, 64, 5], [130, 64 + 70, 200], 1, dict(heads=4, kv=4, dim=64, alibi=True, shared=64, window=40, kind="bf16")),
    ([20, 33], [300, 40], 3, dict(heads=8, kv=2, window=400, lo=lambda pos: pos - 30)),
    ([40, 50], [300, 100], 1, dict(heads=4, kv=2, window=2 ** 31 - 1)),
    ([30] * 70, [100] * 70, 1, dict(heads=4, kv=1, window=9)),
    ([33, 9], [64, 128], 1, dict(heads=4, kv=1, window=33, cap=20.0)),
]


@pytest.mark.parametrize("i", range(len(ALONG)))
def test_windows_along_the_path(i):
    sizes, ctx, back, kw = ALONG[i]
    print(f"\n  {sizes[:4]} over {ctx[:4]}, {kw}", flush=True)
    rng = np.random.default_rng(300 + i)
    b = AlongThePath(rng, drafts(rng, sizes, back), lens=[c + n for c, n in zip(ctx, sizes)], **kw)
    with Dev() as d:
        b.run(d, f"case {i}")


@pytest.mark.parametrize("n,ctx,heads,kv,dim,window", [(40, 100, 4, 2, 128, 3), (70, 31, 4, 4, 64, 12), (64, 0, 2, 1, 64, 1)])
def test_windows_along_any_bits(n, ctx, heads, kv, dim, window):
    """bits that are no tree's: the last `window` set ones before the token's own, which may be left out itself"""
    rng = np.random.default_rng(n)
    rows = rng.random((n, n)) < 0.5
    rows[1], rows[n - 1] = False, True
    b = AlongThePath(rng, [rows, rng.random((n, n)) < 0.8], lens=[ctx + n, ctx + n + 300], heads=heads, kv=kv, dim=dim, window=window, kind="bf16")
    with Dev() as d:
        b.run(d, f"{n} tokens")


@pytest.mark.parametrize("sizes,ctx,kw", [([64, 20], [300, 100], dict(heads=4, kv=2, window=7)), ([40], [10], dict(heads=2, kv=1, dim=64, window=39, kind="bf16")),
                                          ([64, 9, 33], [0, 50, 400], dict(heads=4, kv=4, dim=64, window=20, alibi=True))])
def test_a_chain_in_a_window_is_plain_attention(sizes, ctx, kw):
    """a draft without branches sees what mmoe_attn_paged's tokens see; so it does without MMOE_TREE_WINDOW where the window is no shorter than it"""
    rng = np.random.default_rng(len(sizes))
    for more in (0, 64):
        kw = dict(kw, window=kw["window"] + more)
        b = AlongThePath(rng, drafts(rng, sizes, 1), lens=[c + n for c, n in zip(ctx, sizes)], **kw)
        with Dev() as d:
            b.run(d, "as a tree")
            a = b.args
            if more:
                d.write(b.p_out, b.out0); d.write(b.p_lse, b.lse0)
                M.check(d.lib.mmoe_attn_tree(a, b.cache, b.p_bits, b.words), "a window longer than the paths")
                b.check(d, "without the flag")
            d.write(b.p_out, b.out0); d.write(b.p_lse, b.lse0)
            (a.ws, a.ws_bytes), tree_ws = b.plain_ws, (a.ws, a.ws_bytes)
            M.check(d.lib.mmoe_attn_paged(a, b.cache), "plain")
            a.ws, a.ws_bytes = tree_ws
            b.check(d, "plain")


# ---------------------------------------------------------------------------------------------------- limits behind shared positions
@pytest.mark.parametrize("kw", [dict(lo=lambda pos: 90 + (pos % 7) * 30), dict(lo=lambda pos: pos - 20), dict(lo=lambda pos: np.full(len(pos), 1 << 29)), dict(max_q=30), dict(max_q=2),
                                dict(max_len=128), dict(max_len=250), dict(max_len=510), dict(lost=[(0, 3), (0, 20), (1, 12), (2, 33)]), dict(cut=50, pad=7), dict(with_lse=False),
                                dict(window=40), dict(window=250, alibi=True), dict(shared=64, lost=[(0, 0), (0, 3)], cap=20.0)], ids=lambda kw: "-".join(kw))
def test_limits_behind_shared_positions(kw):
    """masks that hide all of the shared positions, or a part; sequences of which some tokens are not served; positions and blocks that are not there"""
    rng = np.random.default_rng(11)
    sizes, ctx = [40, 3, 64], [300, 200, 500]
    b = TreeBatch(rng, drafts(rng, sizes, 6), lens=[c + n for c, n in zip(ctx, sizes)], heads=4, kv=2, kind="bf16", **dict(dict(shared=128), **kw))
    if "lost" in kw:      # the shared positions' blocks are row 0's
        for s in (1, 2):
            b.table[s, :b.shared // b.bs] = b.table[0, :b.shared // b.bs]
    with Dev() as d:
        b.run(d, str(list(kw)))


# ---------------------------------------------------------------------------------------------------- starts and lengths of any value
@pytest.mark.parametrize("heads,kv,shared,window,dim,n", [(64, 1, 0, 0, 128, 60), (8, 2, 0, 100, 128, 60), (4, 4, 64, 0, 64, 60), (4, 2, 0, 2 ** 31 - 1, 64, 72),
                                                          (4, 1, 128, 2 ** 31 - 1, 128, 72)])
def test_starts_and_lengths_of_any_value(heads, kv, shared, window, dim, n):
    """differences of starts that pass 32 bits: no row past the tokens that the call is told of is written, nor anything behind the workspace. The arrays have
    room for 130 tokens more"""
    rng = np.random.default_rng(heads + window % 7)
    most, more = 40, 130
    b = TreeBatch(rng, drafts(rng, [most] + [1] * (n - 1), 5), lens=[most + 200] + [200 + s for s in range(1, n)], heads=heads, kv=kv, dim=dim, shared=shared, window=window, pad=30 + more,
                  cut=most + n - 1 + 30)
    big = 2 ** 31 - 1
    with Dev() as d:
        a = b.upload(d)
        last, lens = most + n - 1, np.array(b.lens, np.int32)
        starts = [[0, big, LEAST, last] * (n // 4) + [last], [big, LEAST] * (n // 2) + [big], [LEAST] * n + [big], [b.cut, LEAST + 7] * (n // 2) + [0], [-1, b.cut - 1, LEAST, b.cut + 9] * (n // 4) + [5],
                  [0] * n + [big]]
        for start in starts:
            for length in (lens, np.full(n, big), np.full(n, LEAST), np.where(np.arange(n) % 2, lens, -lens)):
                d.write(a.qstart, np.array(start[:n + 1], np.int32)); d.write(a.len, np.array(length, np.int32))
                for fill in (0, 0x7f, 0xff):
                    d.write(a.ws, np.full(a.ws_bytes, fill, np.uint8))
                    M.check(d.lib.mmoe_attn_tree(a, b.cache, b.p_bits, b.words), "attention")
                    raw, lse = d.get(b.p_out, b.out0), d.get(b.p_lse, b.lse0)
                    assert (raw[b.cut:] == 0x1234).all() and (lse[b.cut:] == 77.0).all(), (start[:4], length[:2])
                    body = raw[:, 8:8 + heads * (dim + 8)].reshape(b.ntok, heads, dim + 8)
                    assert (raw[:, :8] == 0x1234).all() and (raw[:, 8 + heads * (dim + 8):] == 0x1234).all() and (body[:, :, dim:] == 0x1234).all()
                    assert np.array_equal(d.get(a.ws + a.ws_bytes, b.ws_guard), b.ws_guard), "written behind the workspace"
