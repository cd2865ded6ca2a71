"""Blocks that sequences share, copy and give back (include/maplemoe.h, Part 3) on the card, against plain numpy."""
import ctypes as C

import numpy as np
import pytest

import maplemoe as M
from draft_ref import compact, fork, free_blocks
from paged_ref import Dev

pytestmark = pytest.mark.gpu
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


class Layers:
    """some layers' caches with random bits in them; strides wider than the values, the space between filled too"""

    def __init__(self, d, rng, layers=3, nblocks=20, kv=2, bs=16, dim=128, kind="f16", token_major=False, gap=8):
        self.d, self.nblocks, self.kv, self.bs, self.dim, self.n = d, nblocks, kv, bs, dim, layers
        self.item = np.uint32 if kind == "f32" else np.uint16
        row = dim + gap
        self.shape = (nblocks, bs, kv, row) if token_major else (nblocks, kv, bs, row)
        self.token_major = token_major
        self.host = [[rng.integers(0, 1 << 16, self.shape).astype(self.item) for _ in range(2)] for _ in range(layers)]
        self.at = [[d.put(x) for x in y] for y in self.host]
        self.caches = (M.KvCache * layers)(*(
            M.KvCache(k=k, v=v, block_stride=bs * kv * row, head_stride=row if token_major else bs * row, token_stride=kv * row if token_major else row, nblocks=nblocks,
                      block_size=bs, heads=kv, head_dim=dim, dtype=M.DTYPE[kind]) for k, v in self.at))

    def positions(self, x):
        """[block][position][head][dim]: what the cache holds, without the space between"""
        return (x if self.token_major else x.transpose(0, 2, 1, 3))[..., :self.dim]

    def check(self, want, note=""):
        """want: positions -> positions"""
        for y, p in zip(self.host, self.at):
            for x, q in zip(y, p):
                w = x.copy()
                self.positions(w)[...] = want(self.positions(x))
                assert np.array_equal(self.d.get(q, x), w), note


def table_of(rng, n, width, nblocks):
    ids = rng.permutation(nblocks)[:n * width]
    return ids.reshape(n, width).astype(np.int32)


# ---------------------------------------------------------------------------------------------------- kept positions moved together
@pytest.mark.parametrize("kw,n,length,part", [
    (dict(), 1, 300, 0.3), (dict(layers=24, kv=4), 5, 60, 0.5), (dict(kv=1, dim=8, gap=0), 2, 200, 0.9), (dict(dim=72, kv=3, kind="f32"), 2, 150, 0.2),
    (dict(dim=256, kv=5, kind="f32", token_major=True), 1, 90, 0.7), (dict(layers=128, kv=1, dim=64, bs=32), 3, 70, 0.1), (dict(layers=1, kv=4, token_major=True), 1, 3000, 0.6),
    (dict(layers=1, kv=1, bs=1024, dim=64), 1, 2000, 0.5), (dict(layers=2, kv=16, dim=128, gap=24), 40, 30, 0.4)])
def test_compact(kw, n, length, part):
    print(f"\n  {kw} {n} sequences of up to {length}", flush=True)
    rng = np.random.default_rng(n * 31 + length)
    bs = kw.get("bs", 16)
    width = -(-length // bs) + 1
    with Dev() as d:
        c = Layers(d, rng, nblocks=n * width + 2, **kw)
        table = table_of(rng, n, width, c.nblocks)
        lens = rng.integers(1, length + 1, n)
        lens[0] = length
        lists = [np.sort(rng.permutation(int(x))[:max(1, int(x * part))]) for x in lens]
        if n > 2:
            lists[1] = lists[1][:1]                 # one that stays where it is
            lists[2] = np.arange(3, int(lens[2]))   # all of them do
        count = np.array([len(x) for x in lists], np.int32)
        first = (np.cumsum(count) - count + 3 * np.arange(n)).astype(np.int32)    # with others' entries between
        kept = rng.integers(0, length, int(first[-1] + count[-1])).astype(np.int32)
        for f, x in zip(first, lists):
            kept[f:f + len(x)] = x
        a = M.KvCompact(table=d.put(table), first=d.put(first), count=d.put(count), kept=d.put(kept), nseq=n, width=width, nkept=len(kept))
        M.check(d.lib.mmoe_kv_compact(a, c.caches, c.n), "mmoe_kv_compact")
        c.check(lambda x: compact(x, table, first, count, kept, len(kept), bs), str(kw))


def test_compact_of_entries_that_are_none():
    """negative positions, ones past the table, blocks that are not the cache's, lists that reach past the array, counts below one"""
    rng = np.random.default_rng(4)
    bs, width, n = 16, 4, 8
    with Dev() as d:
        c = Layers(d, rng, nblocks=n * width)
        table = table_of(rng, n, width, c.nblocks)
        table[1, 2], table[2, 0], table[3, 1] = -1, c.nblocks, 2 ** 31 - 1
        kept = np.concatenate([[3, 9, 70, 2 ** 31 - 1], [10, 20, 33, 50], [2, 5, 30, 40], [1, 18, 40, 60], [-4, 1, 7, 9], [0, 5, 6], [4, 6], [60, 61, 62, 63]]).astype(np.int32)
        first = np.array([0, 4, 8, 12, 16, -1, len(kept), len(kept) - 4], np.int32)
        count = np.array([4, 4, 4, 4, 4, 3, 2, 1000], np.int32)
        count[4] = 4
        for cnt in (count, np.where(np.arange(n) % 2 == 0, -5, count).astype(np.int32), np.zeros(n, np.int32)):
            for y, p in zip(c.host, c.at):
                for x, q in zip(y, p):
                    d.write(q, x)
            a = M.KvCompact(table=d.put(table), first=d.put(first), count=d.put(cnt), kept=d.put(kept), nseq=n, width=width, nkept=len(kept))
            M.check(d.lib.mmoe_kv_compact(a, c.caches, c.n), "mmoe_kv_compact")
            c.check(lambda x: compact(x, table, first, cnt, kept, len(kept), bs), "entries that are none")


def test_compact_and_copy_past_32_bits():
    """blocks 2^31 bytes apart"""
    rng = np.random.default_rng(6)
    apart, bs, kv, dim, nb = 1 << 30, 16, 2, 64, 4
    with Dev() as d:
        base = d.room((nb - 1) * apart * 2 + 2 * kv * bs * dim * 2)
        host = rng.integers(0, 1 << 16, (nb, 2, kv, bs, dim)).astype(np.uint16)
        for i in range(nb):
            d.write(base + i * apart * 2, host[i])
        cache = M.KvCache(k=base, v=base + kv * bs * dim * 2, block_stride=apart, head_stride=bs * dim, token_stride=dim, nblocks=nb, block_size=bs, heads=kv, head_dim=dim,
                          dtype=M.BF16)
        table, kept = np.array([[1, 3, 0]], np.int32), np.array([14, 17, 20, 30], np.int32)
        a = M.KvCompact(table=d.put(table), first=d.put(np.zeros(1, np.int32)), count=d.put(np.array([4], np.int32)), kept=d.put(kept), nseq=1, width=3, nkept=4)
        M.check(d.lib.mmoe_kv_compact(a, cache, 1), "compact")
        k = M.KvCopy(copy_from=d.put(np.array([3], np.int32)), copy_to=d.put(np.array([2], np.int32)), ncopy=1)
        M.check(d.lib.mmoe_kv_copy(k, cache, 1), "copy")
        want = np.moveaxis(compact(np.moveaxis(host, 3, 1), table, [0], [4], kept, 4, bs), 1, 3)
        want[2] = want[3]
        for i in range(nb):
            assert np.array_equal(d.get(base + i * apart * 2, host[i]), want[i]), i


# ---------------------------------------------------------------------------------------------------- blocks' contents
@pytest.mark.parametrize("kw,n", [(dict(), 4), (dict(layers=24, kv=4), 9), (dict(kv=1, dim=8, gap=0, bs=1024), 3), (dict(dim=72, kv=3, kind="f32", token_major=True), 5),
                                  (dict(layers=128, dim=64, bs=32), 2), (dict(kv=40, dim=256, kind="f32", layers=1), 1)])
@pytest.mark.parametrize("counts", [True, False])
def test_copy(kw, n, counts):
    print(f"\n  {kw} {n}", flush=True)
    rng = np.random.default_rng(n)
    bs = kw.get("bs", 16)
    with Dev() as d:
        c = Layers(d, rng, nblocks=2 * n + 3, **kw)
        ids = rng.permutation(c.nblocks)
        src, dst = ids[:n].astype(np.int32), ids[n:2 * n].astype(np.int32)
        src, dst = np.append(src, [-1, src[0], 2 ** 31 - 1]).astype(np.int32), np.append(dst, [dst[0], -1, ids[-1]]).astype(np.int32)   # pairs of which one is none
        count = rng.integers(0, bs + 1, n + 3).astype(np.int32)
        count[0] = -3 if n > 2 else bs + 100
        a = M.KvCopy(copy_from=d.put(src), copy_to=d.put(dst), copy_count=d.put(count) if counts else None, ncopy=n + 3)
        M.check(d.lib.mmoe_kv_copy(a, c.caches, c.n), "mmoe_kv_copy")

        def want(x):
            y = x.copy()
            for i in range(n):
                k = min(max(int(count[i]), 0), bs) if counts else bs
                y[dst[i], :k] = x[src[i], :k]
            return y
        c.check(want, str(kw))


# ---------------------------------------------------------------------------------------------------- copies of sequences, blocks given back
def sequences(rng, n, width, bs, shared=0, spare=40):
    """lengths, a table of their blocks (the first shared ones the same in every row), the free list"""
    keep = shared // bs
    ctx = shared + rng.integers(0, width * bs - shared + 1, n)
    held = -(-ctx // bs)
    nblocks = keep + int((held - keep).sum()) + spare
    ids = rng.permutation(nblocks).astype(np.int32)
    table, at = np.full((n, width), -1, np.int32), keep
    table[:, :keep] = ids[:keep]
    for s in range(n):
        table[s, keep:held[s]] = ids[at:at + held[s] - keep]
        at += held[s] - keep
    free = np.full(nblocks, -5, np.int32)
    free[:nblocks - at] = ids[at:]
    return ctx.astype(np.int32), table, free, nblocks - at, nblocks


def run_fork(src, dst, at, ctx, table, holders, free, nfree, bs, shared, nblocks, in_place, rows_out=None):
    n, width = table.shape
    i = lambda v: np.array(v, np.int32)  # noqa: E731
    ctx_out, table_out = (ctx, table) if in_place else (np.full(n, -3, np.int32), np.full(table.shape, -9, np.int32))
    want = fork(src, dst, at, ctx, ctx_out, table, table_out, holders, free, nfree, bs, shared, nblocks)
    with Dev() as d:
        p_ctx, p_table, z = d.put(ctx), d.put(table), np.full(max(len(src), 1), -99, np.int32)
        p_nfree = d.put(i([nfree]))
        out = dict(ctx_out=p_ctx if in_place else d.put(ctx_out), table_out=p_table if in_place else d.put(table_out), holders=d.put(holders),
                   nfree_out=p_nfree if in_place else d.put(i([0])), copy_from=d.put(z), copy_to=d.put(z), copy_count=d.put(z))
        a = M.KvFork(src=d.put(i(src)), dst=d.put(i(dst)), at=None if at is None else d.put(i(at)), ctx=p_ctx, table=p_table, free_list=d.put(free), nfree=p_nfree, nfork=len(src),
                     nseq=n, width=width, nblocks=nblocks, block_size=bs, shared=shared, **out)
        M.check(d.lib.mmoe_kv_fork(a), "mmoe_kv_fork")
        for k, p in out.items():
            assert np.array_equal(d.get(p, want[k]), want[k]), k
    return want


def run_free(ctx, keep, table, holders, free, nfree, bs, shared, nblocks, in_place):
    n, width = table.shape
    i = lambda v: np.array(v, np.int32)  # noqa: E731
    want = free_blocks(ctx, keep, table, holders, free, nfree, bs, shared, nblocks)
    with Dev() as d:
        for _ in range(2):   # the list comes out the same whatever order the atomics had
            p_ctx, p_nfree = d.put(ctx), d.put(i([nfree]))
            out = dict(len=p_ctx if in_place else d.put(np.full(n, -3, np.int32)), free_list=d.put(free), nfree_out=p_nfree if in_place else d.put(i([0])))
            if holders is not None:
                out["holders"] = d.put(holders)
            a = M.KvFree(ctx=p_ctx, keep=d.put(i(keep)), table=d.put(table), nfree=p_nfree, nseq=n, width=width, nblocks=nblocks, block_size=bs, shared=shared, **out)
            M.check(d.lib.mmoe_kv_free(a), "mmoe_kv_free")
            for k, p in out.items():
                assert np.array_equal(d.get(p, want[k]), want[k]), k
    return want


@pytest.mark.parametrize("n,width,bs,shared,copies,in_place", [(1, 4, 16, 0, 1, True), (3, 40, 16, 0, 5, False), (7, 9, 1024, 1024, 2, True), (16, 130, 32, 64, 4, False),
                                                               (300, 30, 16, 0, 4, False), (2, 2000, 16, 32, 3, True), (900, 3, 16, 16, 4, False)])
def test_fork_then_free(n, width, bs, shared, copies, in_place):
    """copies of some sequences at all and at shorter lengths; then shortened and ended ones among those that share"""
    print(f"\n  {n} sequences, {copies} copies, width {width}", flush=True)
    rng = np.random.default_rng(n * 13 + width)
    ctx, table, free, nfree, nblocks = sequences(rng, n, width, bs, shared, spare=n * copies + 9)
    if in_place:       # rows behind the sequences' for the copies
        rows = n * (copies + 1)
        t, c = np.full((rows, width), -1, np.int32), np.zeros(rows, np.int32)
        t[:n], c[:n] = table, ctx
        src, dst = np.repeat(np.arange(n), copies), n + rng.permutation(n * copies)
    else:
        t, c, rows = np.repeat(table, copies, 0), np.repeat(ctx, copies), n * copies
        src, dst = rng.integers(0, rows, rows), rng.permutation(rows)
    holders = np.zeros(nblocks, np.int32)
    at = np.where(rng.random(len(src)) < 0.5, 1 << 30, rng.integers(0, width * bs + 1, len(src)))
    run_fork(src, dst, None, c, t, holders, free, nfree, bs, shared, nblocks, in_place)
    w = run_fork(src, dst, at, c, t, holders, free, nfree, bs, shared, nblocks, in_place)
    if len(src) > 3:
        run_fork(src, dst, at, c, t, holders, free, 2, bs, shared, nblocks, in_place)       # blocks for two
        run_fork(src, dst, at, c, t, holders, free, -1, bs, shared, nblocks, in_place)
    # what the forks left, given back: some whole, some in part
    t2, c2, h2 = w["table_out"], np.maximum(w["ctx_out"], 0), w["holders"]
    for keep in (np.zeros(rows), np.where(rng.random(rows) < 0.5, 0, rng.integers(0, width * bs + 1, rows)), np.full(rows, 1 << 30), np.maximum(c2 - rng.integers(0, 3 * bs, rows), -5)):
        run_free(c2, keep.astype(np.int64), t2, h2, free, int(w["nfree_out"][0]), bs, shared, nblocks, in_place)
    r = run_free(c2, np.maximum(c2 - bs, 0), t2, None, free, int(w["nfree_out"][0]), bs, shared, nblocks, not in_place)
    assert r["nfree_out"][0] >= w["nfree_out"][0]


def test_everything_comes_back():
    """sequences, their copies, the copies' copies: with the last of them every block is on the list again"""
    rng = np.random.default_rng(12)
    ctx, table, free, nfree, nblocks = sequences(rng, 8, 20, 16, 0, 60)
    rows = 24
    t, c = np.full((rows, 20), -1, np.int32), np.zeros(rows, np.int32)
    t[:8], c[:8] = table, ctx
    h = np.zeros(nblocks, np.int32)
    w = run_fork(np.arange(8), 8 + np.arange(8), None, c, t, h, free, nfree, 16, 0, nblocks, True)
    w = run_fork(8 + np.arange(8), 16 + np.arange(8), None, w["ctx_out"], w["table_out"], w["holders"], free, int(w["nfree_out"][0]), 16, 0, nblocks, True)
    n, free, c, h = int(w["nfree_out"][0]), free, w["ctx_out"], w["holders"]
    for part in (rng.permutation(rows)[:9], np.arange(rows)):
        keep = c.copy()
        keep[part] = 0
        r = run_free(c, keep, w["table_out"], h, free, n, 16, 0, nblocks, False)
        c, h, free, n = r["len"], r["holders"], r["free_list"], int(r["nfree_out"][0])
    assert n == nblocks and sorted(free.tolist()) == list(range(nblocks)) and not h.any()


def test_many_blocks_given_back():
    """far more blocks than a workgroup holds, shared by many; 4096 sequences"""
    rng = np.random.default_rng(2)
    ctx, table, free, nfree, nblocks = sequences(rng, 40, 900, 16, 32, 100)
    t, c = np.repeat(table, 3, 0), np.repeat(ctx, 3)
    h = np.zeros(nblocks, np.int32)
    for row in t[::3]:
        h[row[row >= 0]] = 2
    keep = np.where(rng.random(120) < 0.3, c // 2 // 16 * 16, 0)
    run_free(c, keep, t, h, free, nfree, 16, 32, nblocks, False)
    run_free(c[::3].copy(), keep[::3], table, None, free, nfree, 16, 32, nblocks, True)
    ctx, table, free, nfree, nblocks = sequences(rng, 4096, 5, 16, 0, 100)
    run_free(ctx, rng.integers(0, 80, 4096), table, np.zeros(nblocks, np.int32), free, nfree, 16, 0, nblocks, True)
    run_free(ctx, np.zeros(4096), table, None, free, nfree, 16, 0, nblocks, True)


def test_pages_that_are_none():
    """rows and blocks that are not there, lengths below zero and past the table, a list that claims more than it holds"""
    rng = np.random.default_rng(3)
    ctx, table, free, nfree, nblocks = sequences(rng, 6, 8, 16, 16, 30)
    ctx[0], ctx[1] = 2 ** 31 - 1, -7
    table[2, 3], table[3, 1], table[0, 7] = -1, nblocks, 2 ** 31 - 1
    h = np.zeros(nblocks, np.int32)
    out = run_fork([0, 1, -1, 2, 6, 3, 4], [0, 1, 2, 3, 4, -5, 5], None, ctx, table, h, free, nfree, 16, 16, nblocks, False)
    assert out["copy_from"].max() < nblocks
    run_fork([2, 3], [4, 5], [-3, 2 ** 31 - 1], ctx, table, h, free, 2 ** 31 - 1, 16, 16, nblocks, False)
    run_free(ctx, np.array([0, 5, 20, 9, 2 ** 31 - 1, -2 ** 31]), table, h, free, nfree, 16, 16, nblocks, False)
    run_free(ctx, np.zeros(6), table, None, free, 2 ** 31 - 1, 16, 16, nblocks, True)
    run_free(ctx, np.zeros(6), table, None, free, nblocks - 2, 16, 0, nblocks, True)     # no room in the list for all
    t = table.copy()
    t[4:] = t[4]                          # the same blocks twice without holders that say so: each goes back once
    run_free(np.full(6, 100, np.int32), np.zeros(6), t, h, free, nfree, 16, 16, nblocks, False)
    # nothing to do
    with Dev() as d:
        nf, out = d.put(np.array([7], np.int32)), d.put(np.array([-1], np.int32))
        M.check(d.lib.mmoe_kv_free(M.KvFree(nfree=nf, nfree_out=out, free_list=d.room(400), nseq=0, width=1, nblocks=9, block_size=16)), "free")
        assert d.get(out, np.zeros(1, np.int32))[0] == 7
        M.check(d.lib.mmoe_kv_fork(M.KvFork(nfree=nf, nfree_out=out, nfork=0, nseq=0, width=1, nblocks=0, block_size=16)), "fork")
        assert d.get(out, np.zeros(1, np.int32))[0] == 0      # a cache without blocks has none free


def test_captured_fork_copy_free():
    """a beam search's step captured and replayed over changing parents, with eager calls between"""
    rng = np.random.default_rng(9)
    n, width, bs, steps = 6, 6, 16, 7
    hip = C.CDLL("libamdhip64.so")
    with Dev() as d:
        nblocks = 60
        c = Layers(d, rng, nblocks=nblocks, layers=2)
        ctx = np.full(n, 40, np.int32)
        table = np.full((n, width), -1, np.int32)
        table[:, :3] = np.arange(n * 3).reshape(n, 3)
        free, nfree, holders = np.full(nblocks, -1, np.int32), nblocks - 3 * n, np.zeros(nblocks, np.int32)
        free[:nfree] = np.arange(3 * n, nblocks)
        i = lambda v: np.array(v, np.int32)  # noqa: E731
        p = dict(ctx=d.put(ctx), table=d.put(table), ctx2=d.put(ctx), table2=d.put(table), holders=d.put(holders), free=d.put(free), nfree=d.put(i([nfree])), src=d.put(i(range(n))),
                 dst=d.put(i(range(n))), zero=d.put(i([0] * n)), f=d.put(ctx), t=d.put(ctx), k=d.put(ctx), old=d.put(ctx))
        pages = dict(nseq=n, width=width, nblocks=nblocks, block_size=bs)
        f = M.KvFork(src=p["src"], dst=p["dst"], ctx=p["ctx"], table=p["table"], ctx_out=p["ctx2"], table_out=p["table2"], holders=p["holders"], free_list=p["free"], nfree=p["nfree"],
                     nfree_out=p["nfree"], copy_from=p["f"], copy_to=p["t"], copy_count=p["k"], nfork=n, **pages)
        k = M.KvCopy(copy_from=p["f"], copy_to=p["t"], copy_count=p["k"], ncopy=n)
        g = M.KvFree(ctx=p["ctx"], keep=p["zero"], table=p["table"], nfree=p["nfree"], len=p["old"], free_list=p["free"], nfree_out=p["nfree"], holders=p["holders"], **pages)

        def queue():
            M.check(d.lib.mmoe_kv_fork(f), "fork")
            M.check(d.lib.mmoe_kv_copy(k, c.caches, c.n), "copy")
            M.check(d.lib.mmoe_kv_free(g), "free")

        def text(t, x):    # what each row holds
            return [np.concatenate([x[t[s, j // bs], j % bs][None] for j in range(40)]) for s in range(n)]

        stream, graph, ex = C.c_void_p(d.lib.mmoe_stream()), C.c_void_p(), C.c_void_p()
        assert hip.hipStreamBeginCapture(stream, 1) == 0
        queue()
        assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
        assert hip.hipGraphInstantiate(C.byref(ex), graph, None, None, C.c_size_t(0)) == 0
        try:
            for step in range(steps):
                src = rng.integers(0, n, n)
                d.write(p["src"], i(src))
                before = [[text(table, c.positions(d.get(q, x))) for x, q in zip(y, z)] for y, z in zip(c.host, c.at)]
                if step % 3 == 2:
                    queue()
                else:
                    assert hip.hipGraphLaunch(ex, stream) == 0
                new, h, left = d.get(p["table2"], table), d.get(p["holders"], holders), int(d.get(p["nfree"], i([0]))[0])
                assert (d.get(p["ctx2"], ctx) == 40).all()
                for l in range(c.n):
                    for w in range(2):
                        now = text(new, c.positions(d.get(c.at[l][w], c.host[l][w])))
                        assert all(np.array_equal(now[s], before[l][w][src[s]]) for s in range(n)), (step, l, w)
                used, times = np.unique(new[:, :3], return_counts=True)
                assert np.array_equal(h[used], times - 1) and left == nblocks - len(used), step
                assert sorted(d.get(p["free"], free)[:left].tolist() + used.tolist()) == list(range(nblocks)), step
                table = new
                d.write(p["table"], new)
        finally:
            hip.hipGraphExecDestroy(ex); hip.hipGraphDestroy(graph)


def test_profile_counts_pages():
    with Dev() as d:
        nf = d.put(np.array([0], np.int32))
        ms, cnt = C.c_double(), C.c_long()
        M.check(d.lib.mmoe_prof_reset(), "reset"); M.check(d.lib.mmoe_prof(1), "prof")
        try:
            M.check(d.lib.mmoe_kv_free(M.KvFree(nfree=nf, nfree_out=nf, free_list=nf, nseq=0, width=1, nblocks=1, block_size=16)), "free")
        finally:
            M.check(d.lib.mmoe_prof(0), "prof off")
        M.check(d.lib.mmoe_prof_get(M.KERNELS.index("kv_pages"), C.byref(ms), C.byref(cnt)), "get")
        assert cnt.value == 1 and 0 < ms.value < 50
