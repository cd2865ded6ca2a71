"""Drafted tokens and shared blocks (include/maplemoe.h, Part 3) in plain numpy, one item after the other, as the header words them."""
import numpy as np

import maplemoe as M
from paged_ref import HALF, Batch, attend, decode


def tree(rng, n, back):
    """parents of n nodes, each one of the `back` before it"""
    return [-1 if i == 0 else int(rng.integers(max(0, i - back), i)) for i in range(n)]


def paths(parent):
    """[node][node]: is it the node itself or one that it follows"""
    n = len(parent)
    a = np.zeros((n, n), bool)
    for i, p in enumerate(parent):
        if 0 <= p < i:
            a[i] = a[p]
        a[i, i] = True
    return a


def words_of(rows, words):
    """truth values [token][node] -> bits[token][words]"""
    out = np.zeros((len(rows), words), np.uint64)
    for t, r in enumerate(rows):
        for j in np.nonzero(r)[0]:
            if j < 64 * words:
                out[t, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return out


def tree_plan(qstart, length, parent, words, ntok):
    pos, bits = np.zeros(ntok, np.int32), np.zeros((ntok, words), np.uint64)
    for s in range(len(length)):
        t0, t1 = qstart[s], qstart[s + 1]
        n = min(t1 - t0, 64 * words)
        a = paths(parent[t0:t0 + n])
        bits[t0:t0 + n] = words_of(a, words)
        pos[t0:t0 + n] = length[s] - (t1 - t0) + a.sum(1) - 1
    return pos, bits


def accept(qstart, length, parent, token, choice, kept):
    kept, count, ctx, last = kept.copy(), [], [], []
    for s in range(len(length)):
        t0, n = qstart[s], qstart[s + 1] - qstart[s]
        path = [0] if n else []
        while path:
            i = path[-1]
            follow = [j for j in range(i + 1, min(n, M.TREE_MAX)) if parent[t0 + j] == i and token[t0 + j] == choice[t0 + i]]
            if not follow:
                break
            path.append(follow[0])
        for j, i in enumerate(path):
            kept[t0 + j] = length[s] - n + i
        count.append(len(path)); ctx.append(length[s] - n + len(path)); last.append(choice[t0 + path[-1]] if path else -1)
    i = lambda v: np.array(v, np.int32)  # noqa: E731
    return kept, i(count), i(ctx), i(last)


def compact(cache, table, first, count, kept, nkept, bs):
    """cache [...][block][position][...] with the blocks on axis 0 and positions on axis 1"""
    old, new = cache, cache.copy()
    nblocks, width = cache.shape[0], table.shape[1]
    for s in range(len(first)):
        if not 0 <= first[s] < nkept:
            continue
        k = kept[first[s]:min(int(first[s]) + max(int(count[s]), 0), nkept)].astype(np.int64)
        for j in range(1, len(k)):
            a, b = int(k[j]), int(k[0]) + j
            if a <= b or b < 0 or a >= width * bs:
                continue
            x, y = table[s, a // bs], table[s, b // bs]
            if 0 <= x < nblocks and 0 <= y < nblocks:
                new[y, b % bs] = old[x, a % bs]
    return new


def fork(src, dst, at, ctx, ctx_out, table, table_out, holders, free, nfree, bs, shared, nblocks):
    nseq, width = table.shape
    ctx_out, table_out, holders = ctx_out.copy(), table_out.copy(), holders.copy()
    n = min(max(int(nfree), 0), nblocks)
    f, t, c = (np.full(len(src), v, np.int32) for v in (-1, -1, 0))
    open_ = True
    for i, (a, b) in enumerate(zip(src, dst)):
        ok = 0 <= a < nseq and 0 <= b < nseq
        if not ok:
            if 0 <= b < nseq:
                ctx_out[b] = 0
            continue
        m = int(ctx[a]) if at is None else min(int(ctx[a]), int(at[i]))
        m = min(max(m, 0), width * bs)
        need = m % bs and m > shared
        if need and n == 0:
            open_ = False
        if not open_:
            ctx_out[b] = 0
            continue
        ctx_out[b] = m
        for j in range(-(-m // bs) if m <= shared else m // bs):
            x = table[a, j]
            table_out[b, j] = x
            if j >= shared // bs and 0 <= x < nblocks:
                holders[x] += 1
        if need:
            n -= 1
            table_out[b, m // bs] = free[n]
            f[i], t[i], c[i] = table[a, m // bs], free[n], m % bs
    return dict(ctx_out=ctx_out, table_out=table_out, holders=holders, nfree_out=np.array([n], np.int32), copy_from=f, copy_to=t, copy_count=c)


def free_blocks(ctx, keep, table, holders, free, nfree, bs, shared, nblocks):
    nseq, width = table.shape
    free, n = free.copy(), min(max(int(nfree), 0), nblocks)
    more = None if holders is None else holders.copy()
    length, gives = [], []
    for s in range(nseq):
        c = min(max(int(ctx[s]), 0), width * bs)
        k = min(c, max(int(keep[s]), shared))
        b = table[s, k // bs] if k < c else -1
        if holders is not None and k < c and k % bs and k > shared and 0 <= b < nblocks and holders[b] > 0:
            k = c
        length.append(k)
        gives += [table[s, j] for j in range(max(-(-k // bs), shared // bs), -(-c // bs))]
    last = {b: i for i, b in enumerate(gives)}
    for i, b in enumerate(gives):
        if not 0 <= b < nblocks:
            continue
        if more is not None:
            more[b] -= 1
            if last[b] > i or more[b] >= 0:
                continue
            more[b] = 0
        if n < nblocks:
            free[n] = b
            n += 1
    out = dict(len=np.array(length, np.int32), free_list=free, nfree_out=np.array([n], np.int32))
    return out if holders is None else dict(out, holders=more)


class TreeBatch(Batch):
    """A batch whose new tokens are drafts. rows: per sequence [token][node] truth values, bits past the token itself among them where a test
    wants some (they count for nothing)."""

    def __init__(self, rng, rows, words=None, **kw):
        super().__init__(rng, qlens=[len(r) for r in rows], **kw)
        self.rows = rows
        self.words = words or max(1, -(-max(len(r) for r in rows) // 64))
        every = [row for r in rows for row in r]
        self.bits = np.concatenate([words_of(every, self.words), np.full((self.pad, self.words), (1 << 64) - 1, np.uint64)])

    def expect(self):
        out = np.zeros((self.ntok, self.heads, self.dim))
        lse, off, loff = np.zeros((self.ntok, self.heads)), np.zeros(out.shape), np.zeros((self.ntok, self.heads))
        q = decode(self.q, self.kind)
        for s, rows in enumerate(self.rows):
            k, v = self.cached(s)
            n = len(rows)
            ctx = self.lens[s] - n
            b = self.table[s][np.arange(self.lens[s]) // self.bs]
            there = (b >= 0) & (b < self.nblocks) & (np.arange(self.lens[s]) < self.max_len)
            for i, row in enumerate(rows):
                t = self.qstart[s] + i
                # the cached positions, then the path: one behind the other, so that a place in this list is a position
                chain = list(range(ctx)) + [ctx + j for j in range(i) if row[j]] + [ctx + i]
                pos = len(chain) - 1
                see = there[chain]
                see[-1] &= bool(row[i])
                lo = 0 if self.lo is None else int(self.lo[t])
                if self.window:
                    lo = max(lo, pos - self.window)
                see[:ctx] &= np.arange(ctx) >= lo
                with np.errstate(all="ignore"):
                    o, l, e, f = attend(q[t:t + 1], k[chain], v[chain], np.array([pos]), see[None], self.scale, self.cap, self.slopes, HALF[self.kind])
                out[t], lse[t], off[t], loff[t] = o[0], l[0], e[0], f[0]
        return out, lse, off, loff

    def upload(self, d):
        a = super().upload(d)
        self.p_bits = d.put(self.bits)
        self.plain_ws = a.ws, a.ws_bytes
        size = d.lib.mmoe_attn_tree_ws(a, self.cache, self.p_bits, self.words)
        assert size, d.lib.mmoe_last_error()
        a.ws, a.ws_bytes = d.room(size + 256), size
        d.write(a.ws + size, self.ws_guard)
        return a

    def run(self, d, note=""):
        a = self.upload(d)
        M.check(d.lib.mmoe_attn_tree(a, self.cache, self.p_bits, self.words), "mmoe_attn_tree")
        return self.check(d, note)
