"""The many-sequence operators (include/maplemoe.h, Part 3) in plain numpy, in 64 bits, and device buffers for their tests."""
import ctypes as C

import numpy as np

import maplemoe as M

HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}   # half a step of rounding, relative to the value


def encode(x, kind):
    """float array -> the type's bits, rounded to nearest even (float32, or uint16 words)"""
    x = np.ascontiguousarray(x, np.float32)
    if kind == "f32":
        return x
    if kind == "f16":
        return x.astype(np.float16).view(np.uint16)
    u = x.view(np.uint32)
    r = ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7fc0), r)


def decode(b, kind):
    """bits -> float64"""
    if kind == "f32":
        return b.astype(np.float64)
    if kind == "f16":
        return b.view(np.float16).astype(np.float64)
    return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


class Dev:
    """Device copies of numpy arrays, freed together"""

    def __init__(self):
        self.lib, self.held = M.lib(), []

    def __enter__(self):
        return self

    def __exit__(self, *_):
        self.lib.mmoe_sync()
        for p in self.held:
            self.lib.mmoe_dev_free(p)

    def room(self, nbytes):
        p = self.lib.mmoe_dev_alloc(max(int(nbytes), 256))
        assert p, self.lib.mmoe_last_error()
        self.held.append(p)
        return p

    def put(self, a):
        if a is None:
            return None
        a = np.ascontiguousarray(a)
        p = self.room(a.nbytes)
        if a.nbytes:
            M.check(self.lib.mmoe_h2d(p, M.ptr(a), a.nbytes), "h2d")
        return p

    def write(self, p, a):
        a = np.ascontiguousarray(a)
        M.check(self.lib.mmoe_h2d(p, M.ptr(a), a.nbytes), "h2d")

    def get(self, p, like):
        a = np.empty(like.shape, like.dtype)
        if a.nbytes:
            M.check(self.lib.mmoe_d2h(M.ptr(a), p, a.nbytes), "d2h")
        return a


# ---------------------------------------------------------------------------------------------------- block tables
def plan(ctx, add, done, table, free, nfree, bs, shared, ntok, nblocks):
    """one sequence after the other, as the header words it"""
    table, free = table.copy(), free.copy()
    ctx, n, width = list(ctx), min(max(int(nfree), 0), nblocks), table.shape[1]
    keep = shared // bs
    if done is not None:
        for s, d in enumerate(done):
            if d:
                for j in range(keep, -(-min(max(ctx[s], 0), width * bs) // bs)):
                    if n < nblocks:
                        free[n] = table[s, j]
                        n += 1
                ctx[s] = min(ctx[s], shared)
    qstart, length, open_, took = [0], [], True, 0
    for s in range(len(ctx)):
        c, a = int(ctx[s]), int(add[s])
        ok = c >= 0 and a >= 0 and c + a <= width * bs
        need = -(-(c + a) // bs) - -(-c // bs) if ok and a else 0
        if not ok or qstart[-1] + a > ntok or took + need > n:
            open_ = False
        if open_:
            for j in range(need):
                table[s, -(-c // bs) + j] = free[n - 1 - took - j]
            took += need
        length.append(c + (a if open_ else 0))
        qstart.append(qstart[-1] + (a if open_ else 0))
    pos, slot = np.zeros(ntok, np.int32), np.full(ntok, -1, np.int32)
    for s in range(len(ctx)):
        for t in range(qstart[s], qstart[s + 1]):
            pos[t] = length[s] - (qstart[s + 1] - t)
            b = table[s, pos[t] // bs]
            slot[t] = b * bs + pos[t] % bs if 0 <= b < nblocks else -1
    i = lambda v: np.array(v, np.int32)  # noqa: E731
    return dict(table=table, free_list=free, nfree_out=i([n - took]), len=i(length), qstart=i(qstart), pos=pos, slot=slot)


# ---------------------------------------------------------------------------------------------------- rotary positions
def rotate(x, pos, freq, rot, inter, mag):
    """x [n][heads][dim], float64"""
    y = x.copy()
    a = np.outer(pos.astype(np.float64), freq)[:, None]
    c, s = np.cos(a) * mag, np.sin(a) * mag
    i, j = (np.arange(0, rot, 2), np.arange(1, rot, 2)) if inter else (np.arange(rot // 2), np.arange(rot // 2) + rot // 2)
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
    return y


# ---------------------------------------------------------------------------------------------------- attention
def attend(q, keys, values, pos, see, scale, cap, slopes, half):
    """One sequence: q [n][heads][dim], keys / values [len][kv heads][dim] in float64, pos [n], see [n][len]. Returns out, lse and
    how far each may be off: half a step for the result and one for the weights, 32-bit sums for the scores (dim products, each
    within 2^-24 of the sum of their sizes, then a few operations), fp16's smallest step for weights below its normal range."""
    n, heads, dim = q.shape
    g, length = heads // keys.shape[1], keys.shape[0]
    out, lse = np.zeros_like(q), np.full((n, heads), -np.inf)
    off, loff = np.zeros_like(q), np.zeros((n, heads))
    far = np.abs(pos[:, None] - np.arange(length))
    for h in range(heads):
        k, v = keys[:, h // g], values[:, h // g]
        for i in range(n):
            m = see[i]
            if not m.any():
                continue
            km, vm = k[m], v[m]
            with np.errstate(all="ignore"):
                x = km @ q[i, h] * scale
                e = dim * 2.0 ** -24 * (np.abs(km) @ np.abs(q[i, h])) * abs(scale) + 2.0 ** -22 * np.abs(x)
                if cap:
                    x = cap * np.tanh(x / cap)
                    e = e + 2.0 ** -21 * cap
                if slopes is not None:
                    x = x - float(slopes[h]) * far[i][m]
                    e = e + 2.0 ** -22 * abs(float(slopes[h])) * far[i][m]   # the product's size counts, whatever its sign
                top = x.max()
                if top == -np.inf:
                    continue
                if not top < np.inf:     # a score that is NaN or infinite
                    out[i, h], lse[i, h] = np.nan, np.nan
                    continue
                w = np.exp(x - top)
                e = (e + 2.0 ** -22 * np.abs(x - top) + 2.0 ** -21)
                l = w.sum()
                out[i, h] = w @ vm / l
                lse[i, h] = top + np.log(l)
                e = e[w > 1e-30].max()
                size = w @ np.abs(vm) / l
                # fp16 weights, the largest at least 2^7: down to 2^-21 of it they keep half a step, below that they are off by at most 2^-32
                off[i, h] = half * np.abs(out[i, h]) + (half + 2 * e) * size * 1.01 + (2.0 ** -32 * np.abs(vm).sum(0) / l if half == HALF["f16"] else 0) + 2.0 ** -25
                loff[i, h] = e + 2.0 ** -22 * abs(lse[i, h]) + 2.0 ** -20
    return out, lse, off, loff


class Batch:
    """A batch of sequences over a block cache whose unused places hold NaN, with its device arrays, and the reference result."""

    def __init__(self, rng, kind="f16", dim=128, heads=4, kv=1, bs=16, qlens=(1,), lens=(1,), shared=0, window=0, cap=0.0, alibi=False, lo=None,
                 hi=None, pad=0, token_major=False, width_more=2, max_q=None, max_len=None, spread=1.0, poison=None, lost=(), with_lse=True, cut=None):
        self.kind, self.dim, self.heads, self.kv, self.bs, self.qlens, self.lens = kind, dim, heads, kv, bs, list(qlens), list(lens)
        self.shared, self.window, self.cap, self.pad, self.with_lse = shared, window, cap, pad, with_lse
        n, keep = len(lens), shared // bs
        held = [max(keep, -(-x // bs)) for x in lens]
        self.width = max(held + [1]) + width_more
        self.nblocks = keep + sum(h - keep for h in held) + 3
        ids = rng.permutation(self.nblocks)
        self.table = np.full((n, self.width), -1, np.int32)
        self.table[:, :keep] = ids[:keep]
        at = keep
        for s in range(n):
            self.table[s, keep:held[s]] = ids[at:at + held[s] - keep]
            at += held[s] - keep
        shape = (self.nblocks, bs, kv, dim)
        self.k, self.v = (encode(np.full(shape, np.nan), kind) for _ in range(2))
        for s in range(n):
            for p in range(max(lens[s], keep * bs if s == 0 else 0)):
                b = self.table[s, p // bs]
                if p < shared and s:
                    continue
                self.k[b, p % bs] = encode(rng.standard_normal((kv, dim)) * spread, kind)
                self.v[b, p % bs] = encode(rng.standard_normal((kv, dim)), kind)
        if poison:
            poison(self)
        self.qstart = np.concatenate([[0], np.cumsum(self.qlens)]).astype(np.int32)
        self.ntok = int(self.qstart[-1]) + pad
        self.cut = self.ntok if cut is None else cut     # tokens the call is told of
        self.q = encode(rng.standard_normal((self.ntok, heads, dim)) * 1.5, kind)
        self.slopes = (2.0 ** (-8.0 * np.arange(1, heads + 1) / heads)).astype(np.float32) if alibi else None
        self.pos = np.concatenate([np.arange(L - ql, L) for ql, L in zip(self.qlens, lens)] + [np.zeros(pad)]).astype(np.int64)
        self.lo = None if lo is None else np.asarray(lo(self.pos), np.int32)
        self.hi = None if hi is None else np.asarray(hi(self.pos), np.int32)
        for s, j in lost:   # block ids that are not the cache's
            self.table[s, j] = rng.choice([-1, -7, self.nblocks, 2 ** 31 - 1])
        self.max_q = max(self.qlens + [1]) if max_q is None else max_q
        self.max_len = max(lens) if max_len is None else max_len
        self.token_major = token_major
        self.scale = dim ** -0.5

    def sees(self, s):
        t = np.arange(self.qstart[s], self.qstart[s + 1])
        p, pos = np.arange(self.lens[s]), self.pos[t]
        lo = np.zeros(len(t), np.int64) if self.lo is None else self.lo[t].astype(np.int64)
        hi = pos + 1 if self.hi is None else self.hi[t]
        if self.window:
            lo = np.maximum(lo, pos - self.window)
        ok = (p >= lo[:, None]) & (p < hi[:, None]) & (p < self.max_len)
        b = self.table[s][p // self.bs]
        return ok & ((b >= 0) & (b < self.nblocks))[None]

    def cached(self, s):
        p = np.arange(self.lens[s])
        b = self.table[s][p // self.bs]
        b = np.where((b >= 0) & (b < self.nblocks), b, 0)
        return decode(self.k[b, p % self.bs], self.kind), decode(self.v[b, p % self.bs], self.kind)

    def expect(self):
        out = np.zeros((self.ntok, self.heads, self.dim))
        lse, off, loff = np.zeros((self.ntok, self.heads)), np.zeros(out.shape), np.zeros((self.ntok, self.heads))
        q = decode(self.q, self.kind)
        for s in range(len(self.lens)):
            t = slice(self.qstart[s], self.qstart[s + 1])
            k, v = self.cached(s)
            with np.errstate(all="ignore"):
                out[t], lse[t], off[t], loff[t] = attend(q[t], k, v, self.pos[t], self.sees(s), self.scale, self.cap, self.slopes, HALF[self.kind])
        return out, lse, off, loff

    def upload(self, d):
        """device arrays and the argument blocks; q lies inside wider rows, the head strides differ from dense ones"""
        n, h, dim, e = self.ntok, self.heads, self.dim, 2
        self.qrow, self.orow = h * dim + 24, h * (dim + 8) + 16
        qw = encode(np.full((n, self.qrow), np.nan), self.kind)
        qw[:, 8:8 + h * dim] = self.q.reshape(n, -1)
        self.out0 = np.full((n, self.orow), 0x1234, np.uint16)
        self.lse0 = np.full((n, h), 77.0, np.float32)
        c = [x if self.token_major else x.transpose(0, 2, 1, 3) for x in (self.k, self.v)]
        block = self.bs * self.kv * dim
        self.cache = M.KvCache(k=d.put(c[0]), v=d.put(c[1]), block_stride=block, head_stride=dim if self.token_major else self.bs * dim,
                               token_stride=self.kv * dim if self.token_major else dim, nblocks=self.nblocks, block_size=self.bs, heads=self.kv,
                               head_dim=dim, dtype=M.DTYPE[self.kind])
        self.p_out, self.p_lse = d.put(self.out0), d.put(self.lse0)
        a = M.PagedAttn(q=d.put(qw) + 8 * e, out=self.p_out + 16, lse=self.p_lse if self.with_lse else None, q_token=self.qrow, q_head=dim, out_token=self.orow,
                        out_head=dim + 8, qstart=d.put(self.qstart), len=d.put(np.array(self.lens, np.int32)), table=d.put(self.table), lo=d.put(self.lo),
                        hi=d.put(self.hi), slopes=d.put(self.slopes), nseq=len(self.lens), ntok=self.cut, heads=h, width=self.width, max_q=self.max_q,
                        max_len=self.max_len, shared=self.shared, window=self.window, scale=self.scale, cap=self.cap)
        size = d.lib.mmoe_attn_paged_ws(a, self.cache)
        assert size, d.lib.mmoe_last_error()
        self.ws_guard = np.full(256, 0x5a, np.uint8)
        a.ws, a.ws_bytes = d.room(size + 256), size
        d.write(a.ws + size, self.ws_guard)
        self.args = a
        return a

    def check(self, d, note=""):
        """what the device holds against the reference; everything around it untouched"""
        out, lse, off, loff = self.expect()
        raw = d.get(self.p_out, self.out0)
        n, h, dim = self.ntok, self.heads, self.dim
        body = raw[:, 8:8 + h * (dim + 8)].reshape(n, h, dim + 8)
        live = int(self.qstart[-1])
        got = decode(body[:live, :, :dim].copy(), self.kind)
        served = np.zeros(n, bool)
        for s in range(len(self.lens)):
            served[self.qstart[s]:min(self.qstart[s + 1], self.qstart[s] + self.max_q)] = True
        served[self.cut:] = False
        assert (raw[:, :8] == 0x1234).all() and (raw[:, 8 + h * (dim + 8):] == 0x1234).all() and (body[:, :, dim:] == 0x1234).all(), "written beside the rows"
        assert (raw[~served] == 0x1234).all(), "rows of no token written"
        assert np.array_equal(d.get(self.args.ws + self.args.ws_bytes, self.ws_guard), self.ws_guard), "written behind the workspace"
        sv = served[:live]
        fin = np.isfinite(out[:live])
        assert np.array_equal(np.isnan(got)[sv], np.isnan(out[:live])[sv]), f"NaN at other places {note}"
        same = ~fin & ~np.isnan(out[:live])
        got, out = np.where(sv[:, None, None], got, 0), np.where(served[:, None, None], out, 0)
        assert np.array_equal(got[same & sv[:, None, None]], out[:live][same & sv[:, None, None]])
        fin &= sv[:, None, None]
        got, out = np.where(fin, got, 0), np.where(fin, out[:live], 0)
        bad = np.abs(got - out) > off[:live]
        worst = (np.abs(got - out)[fin] / np.maximum(off[:live][fin], 1e-30)).max() if fin.any() else 0.0
        print(f"  {note}: {live} tokens, error at most {worst:.2f} of the bound", flush=True)
        assert not bad.any(), (note, np.argwhere(bad)[:5], got[bad][:5], out[bad][:5])
        if self.with_lse:
            gl = d.get(self.p_lse, self.lse0)
            assert (gl[~served] == 77.0).all()
            gl, l, lo = gl[:live][sv].astype(np.float64), lse[:live][sv], loff[:live][sv]
            f = np.isfinite(l)
            assert np.array_equal(gl[l == -np.inf], l[l == -np.inf]) and not np.isfinite(gl[np.isnan(l)]).any()
            gl, l, lo = gl[f], l[f], lo[f]
            assert (np.abs(gl - l) <= lo).all(), (note, "lse", np.abs(gl - l).max())
        return worst
