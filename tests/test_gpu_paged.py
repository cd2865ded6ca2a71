"""The operators that serve many sequences at once (include/maplemoe.h, Part 3) on the card, against plain numpy in 64 bits."""
import ctypes as C

import numpy as np
import pytest

import maplemoe as M
from paged_ref import HALF, Batch, Dev, decode, encode, plan, rotate

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------------- block tables
def make_plan(rng, n, ctx, add, bs, width, nblocks, shared=0, done=None, nfree=None, ntok=None):
    ctx, add = np.array(ctx, np.int32), np.array(add, np.int32)
    keep = shared // bs
    ids = rng.permutation(nblocks).astype(np.int32)
    table = np.full((n, width), -1, np.int32)
    table[:, :keep] = ids[:keep]
    at = keep
    for s in range(n):
        held = min(-(-max(int(ctx[s]), 0) // bs), width)
        k = max(held - keep, 0)
        table[s, keep:keep + k] = ids[at:at + k]
        at += k
    assert at <= nblocks
    free = np.full(nblocks, -5, np.int32)
    free[:nblocks - at] = ids[at:]
    return dict(ctx=ctx, add=add, done=None if done is None else np.array(done, np.int32), table=table, free=free,
                nfree=nblocks - at if nfree is None else nfree, bs=bs, shared=shared, ntok=int(add.clip(0).sum()) if ntok is None else ntok, nblocks=nblocks)


def run_plan(c, in_place=False):
    n, width = c["table"].shape
    with Dev() as d:
        z = lambda k: np.full(k, -99, np.int32)  # noqa: E731
        ctx, nf = d.put(c["ctx"]), d.put(np.array([c["nfree"]], np.int32))
        held = dict(table=(d.put(c["table"]), c["table"]), free_list=(d.put(c["free"]), c["free"]), nfree_out=(nf if in_place else d.put(z(1)), z(1)),
                    len=(ctx if in_place else d.put(z(n)), z(n)), qstart=(d.put(z(n + 1)), z(n + 1)), pos=(d.put(z(c["ntok"])), z(c["ntok"])),
                    slot=(d.put(z(c["ntok"])), z(c["ntok"])))
        a = M.KvPlan(ctx=ctx, add=d.put(c["add"]), done=d.put(c["done"]), nfree=nf, nseq=n, width=width, nblocks=c["nblocks"], block_size=c["bs"],
                     shared=c["shared"], ntok=c["ntok"], **{k: v[0] for k, v in held.items()})
        M.check(d.lib.mmoe_kv_plan(a), "mmoe_kv_plan")
        return {k: d.get(p, like) for k, (p, like) in held.items()}


def check_plan(c, **kw):
    want = plan(c["ctx"], c["add"], c["done"], c["table"], c["free"], c["nfree"], c["bs"], c["shared"], c["ntok"], c["nblocks"])
    got = run_plan(c, **kw)
    for k in want:
        assert np.array_equal(got[k], want[k]), (k, got[k], want[k])
    return want


@pytest.mark.parametrize("n,bs,add,in_place", [(1, 16, 1, False), (1, 1024, 3000, False), (7, 16, 40, True), (64, 16, 1, False), (301, 64, 90, False),
                                               (1023, 16, 1, True), (1500, 32, 3, False), (4096, 16, 2, True)])
def test_plan_ragged(n, bs, add, in_place):
    print(f"\n  n={n} bs={bs} add={add} in_place={in_place}", flush=True)
    rng = np.random.default_rng(n * 7 + bs)
    ctx, new = rng.integers(0, 5 * bs, n), rng.integers(0, add + 1, n)
    width = int((-(-(ctx + new) // bs)).max()) + 2
    total = int((-(-(ctx + new) // bs)).sum())
    done = (rng.random(n) < 0.2).astype(int) if n > 1 else [1]
    check_plan(make_plan(rng, n, ctx, new, bs, width, total + 9, done=done), in_place=in_place)


def test_plan_shared_prefix_and_padding():
    rng = np.random.default_rng(5)
    n, bs, shared = 40, 32, 128
    ctx = shared + rng.integers(0, 200, n)
    ctx[3] = 40          # a row that has not got the whole prefix yet
    new = rng.integers(0, 9, n)
    c = make_plan(rng, n, ctx, new, bs, 20, 700, shared=shared, done=rng.random(n) < 0.3, ntok=int(new.sum()) + 33)
    w = check_plan(c)
    assert (w["slot"][-33:] == -1).all()
    check_plan(dict(c, ntok=9000))     # padded past one workgroup's tokens


@pytest.mark.parametrize("what", ["blocks", "tokens", "width", "negative ctx", "negative add", "no free", "huge add", "list count"])
def test_plan_what_does_not_fit(what):
    print(f"\n  {what}", flush=True)
    rng = np.random.default_rng(11)
    n, bs = 30, 16
    ctx, new = rng.integers(0, 90, n), rng.integers(1, 60, n)
    kw = {}
    if what == "width":
        new[17] = 16 * 40
    if what == "negative add":
        new[12] = -3
    if what == "huge add":
        new[9:12] = 2 ** 31 - 1
    if what == "tokens":
        kw["ntok"] = int(new[:20].sum()) + 3
    c = make_plan(rng, n, ctx, new, bs, 14, 700, done=rng.random(n) < 0.2, **dict(dict(ntok=2000), **kw))
    if what == "negative ctx":
        c["ctx"][8] = -1
    if what == "blocks":
        c["nfree"] = 25
    if what == "no free":
        c["nfree"] = -4
    if what == "list count":
        c["nfree"] = 2 ** 31 - 1     # more than the list holds: as many as it holds
        c["done"] = None
    w = check_plan(c)
    if what not in ("list count",):
        assert w["qstart"][-1] < max(int(new.clip(0, 10 ** 6).sum()), 1)


def test_plan_bad_block_of_a_begun_page_and_empty_batch():
    rng = np.random.default_rng(3)
    c = make_plan(rng, 3, [5, 17, 3], [4, 4, 14], 16, 4, 40)
    c["table"][1, 1] = 40       # not a block of the cache: its tokens have no slot
    c["table"][2, 0] = -1       # the first 13 tokens of the third have none either, its last is in a new block
    w = check_plan(c)
    assert (w["slot"][4:8] == -1).all() and (w["slot"][8:21] == -1).all() and w["slot"][21] >= 0
    with Dev() as d:
        nf, q, out = d.put(np.array([7], np.int32)), d.put(np.array([-1], np.int32)), np.zeros(1, np.int32)
        slot, free = d.put(np.full(5, 3, np.int32)), d.put(np.zeros(9, np.int32))
        a = M.KvPlan(nfree=nf, nfree_out=nf, qstart=q, pos=d.put(np.full(5, 3, np.int32)), slot=slot, free_list=free, nseq=0, width=1, nblocks=9, block_size=16, ntok=5)
        M.check(d.lib.mmoe_kv_plan(a), "empty batch")
        assert d.get(nf, out)[0] == 7 and d.get(q, out)[0] == 0 and (d.get(slot, np.zeros(5, np.int32)) == -1).all()


# ---------------------------------------------------------------------------------------------------- rotary positions
ROPES = [  # tokens, heads, kv heads, head_dim, rot, interleaved, in, out, block size (0: no cache), token-major cache, far
    (1, 16, 4, 128, 64, 0, "f32", "f16", 16, False, 4096),
    (64, 16, 4, 128, 128, 1, "f16", "f16", 32, True, 4096),
    (37, 3, 1, 64, 20, 0, "bf16", "bf16", 16, False, 1000000),
    (37, 3, 1, 64, 20, 1, "bf16", "bf16", 16, True, 1000000),
    (130, 12, 12, 64, 64, 0, "f32", "bf16", 64, False, 100000),
    (2100, 5, 1, 24, 2, 0, "f16", "f32", 0, False, 9),
    (300, 6, 2, 256, 256, 0, "f32", "f32", 1024, False, 200000),
    (8200, 2, 1, 72, 70, 0, "f16", "f16", 16, False, 50000),
    (9001, 2, 2, 128, 0, 0, "bf16", "bf16", 64, False, 50000),
    (50, 0, 2, 128, 32, 1, "f32", "f16", 16, False, 500),
    (50, 4, 0, 128, 32, 0, "f32", "f16", 0, False, 500),
]


@pytest.mark.parametrize("n,heads,kv,dim,rot,inter,tin,tout,bs,token_major,far", ROPES)
def test_rope(n, heads, kv, dim, rot, inter, tin, tout, bs, token_major, far):
    print(f"\n  n={n} heads={heads}/{kv} dim={dim} rot={rot} inter={inter} {tin}->{tout} bs={bs}", flush=True)
    rng = np.random.default_rng(n + dim + rot)
    freq = np.zeros(max(rot // 2, 1))
    M.check(M.lib().mmoe_rope_freqs(rot, 10000.0, 4.0, 2048, 1.0, 32.0, M.ptr(freq)), "freqs")
    row = (heads + 2 * kv) * dim + 16
    x = rng.standard_normal((n, row)).astype(np.float32)
    xe = encode(x, tin)
    part = lambda a, b: decode(np.ascontiguousarray(xe[:, a * dim:b * dim]), tin).reshape(n, b - a, dim)  # noqa: E731
    pos = rng.integers(0, far, n).astype(np.int32)
    pos[0] = far
    mag = np.float32(1.1)
    q, k, v = rotate(part(0, heads), pos, freq, rot, inter, float(mag)), rotate(part(heads, heads + kv), pos, freq, rot, inter, float(mag)), part(heads + kv, heads + 2 * kv)
    # half a step of the result; 32-bit cos, sin and products: 2^-21 of the pair's size (mag * 1.42 * |x|), for the angle's 32-bit half turns included
    def off(y, big):
        return HALF[tout] * np.abs(y) + 2.0 ** -20 * np.abs(big).max() * 1.6 + 2.0 ** -25
    with Dev() as d:
        size = 4 if tin == "f32" else 2
        px = d.put(xe)
        q0 = encode(np.full((n, heads, dim + 8), 9.0), tout)
        pq = d.put(q0)
        a = M.Rope(q=px, k=px + heads * dim * size, v=px + (heads + kv) * dim * size, q_out=pq, q_token=row, q_head=dim, k_token=row, k_head=dim, v_token=row,
                   v_head=dim, qo_token=heads * (dim + 8), qo_head=dim + 8, pos=d.put(pos), freq=d.put(freq), ntok=n, heads=heads, kv_heads=kv, head_dim=dim,
                   rot=rot, interleaved=inter, in_dtype=M.DTYPE[tin], out_dtype=M.DTYPE[tout], mag=mag)
        skip = np.zeros(n, bool)
        if bs:
            nblocks = -(-n // bs) + 2
            slot = rng.permutation(nblocks * bs)[:n].astype(np.int32)
            skip = rng.random(n) < 0.1
            slot[skip] = rng.choice([-1, -50, nblocks * bs, 2 ** 31 - 1], skip.sum())
            c0 = encode(np.full((nblocks, bs, kv, dim) if token_major else (nblocks, kv, bs, dim), 5.0), tout)
            pk, pv = d.put(c0), d.put(c0)
            a.slot = d.put(slot)
            cache = M.KvCache(k=pk, v=pv, block_stride=bs * kv * dim, head_stride=dim if token_major else bs * dim, token_stride=kv * dim if token_major else dim,
                              nblocks=nblocks, block_size=bs, heads=kv, head_dim=dim, dtype=M.DTYPE[tout])
            M.check(d.lib.mmoe_rope_kv(a, cache), "rope")
            for p, y, big in ((pk, k, k), (pv, v, v * 0)):
                c = decode(d.get(p, c0), tout)
                c = (c if token_major else c.transpose(0, 2, 1, 3)).reshape(nblocks * bs, kv, dim)
                want = np.full(c.shape, 5.0)
                want[slot[~skip]] = y[~skip]
                tol = np.zeros(c.shape)
                tol[slot[~skip]] = off(y, big)[~skip]
                assert (np.abs(c - want) <= tol).all(), np.abs(c - want).max()
        else:
            k0 = encode(np.full((n, kv, dim), 5.0), tout)
            a.k_out, a.ko_token, a.ko_head = d.put(k0), kv * dim, dim
            M.check(d.lib.mmoe_rope_kv(a, None), "rope")
            if kv:
                assert (np.abs(decode(d.get(a.k_out, k0), tout) - k) <= off(k, k)).all()
        got = decode(d.get(pq, q0), tout).reshape(n, heads, dim + 8)
        assert (got[..., dim:] == 9).all() and (got[skip] == 9).all()
        if heads:
            err = np.abs(got[..., :dim] - q)[~skip]
            assert (err <= off(q, q)[~skip]).all(), err.max()


@pytest.mark.parametrize("rot,inter", [(64, 0), (64, 1), (20, 0), (128, 0)])
def test_rope_in_place_equals_out_of_place(rot, inter):
    print(f"\n  rot={rot} inter={inter}", flush=True)
    rng = np.random.default_rng(rot)
    n, heads, kv, dim = 700, 6, 2, 128
    freq = np.zeros(rot // 2)
    M.check(M.lib().mmoe_rope_freqs(rot, 10000.0, 1.0, 0, 0.0, 0.0, M.ptr(freq)), "freqs")
    x = encode(rng.standard_normal((n, heads + kv, dim)), "bf16")
    row = (heads + kv) * dim
    with Dev() as d:
        got = []
        for same in (False, True):
            px = d.put(x)
            po = px if same else d.put(x * 0)
            a = M.Rope(q=px, k=px + heads * dim * 2, q_out=po, k_out=po + heads * dim * 2, q_token=row, q_head=dim, k_token=row, k_head=dim, qo_token=row, qo_head=dim,
                       ko_token=row, ko_head=dim, pos=d.put(np.arange(n, dtype=np.int32)), freq=d.put(freq), ntok=n, heads=heads, kv_heads=kv, head_dim=dim, rot=rot,
                       interleaved=inter, in_dtype=M.BF16, out_dtype=M.BF16, mag=1.0)
            M.check(d.lib.mmoe_rope_kv(a, None), "rope")
            got.append(d.get(po, x))
        assert np.array_equal(*got) and not np.array_equal(got[0], x)


# ---------------------------------------------------------------------------------------------------- attention
def poison(*where):
    """(sequence, position, k or v, value, dims) written into the cache"""
    def put(b):
        for s, p, which, x, dims in where:
            c = b.k if which == "k" else b.v
            c[b.table[s, p // b.bs], p % b.bs, :, dims] = encode(np.array([x]), b.kind)[0]
    return put


INF, NAN = float("inf"), float("nan")
SOME = slice(3, 9)
ODD = [(0, 250, "v", INF, SOME), (0, 251, "v", NAN, slice(60, 62)), (0, 20, "v", -INF, slice(10, 11)), (0, 290, "v", INF, slice(0, 1)), (0, 291, "v", -INF, slice(0, 1)),
       (1, 128, "v", NAN, slice(0, 64)), (2, 5, "v", INF, slice(63, 64))]
ATTN = {
    "one token, one position": dict(qlens=[1], lens=[1]),
    "one token at block and tile borders": dict(qlens=[1] * 9, lens=[2, 15, 16, 17, 31, 32, 33, 63, 65], heads=16, kv=4),
    "one token, long": dict(qlens=[1], lens=[5000], heads=16, kv=4, kind="bf16", width_more=40),
    "one token each, many sequences": dict(qlens=[1] * 40, lens=[1 + (s * 37) % 400 for s in range(40)], heads=8, kv=2, kind="bf16", bs=32),
    "multi-query heads": dict(qlens=[1, 3, 2], lens=[300, 70, 2], heads=20, kv=1, dim=64),
    "every head its own keys": dict(qlens=[1, 40, 2], lens=[130, 77, 700], heads=3, kv=3, dim=64, kind="bf16"),
    "groups of three, of five, of seven": [dict(qlens=[1, 30], lens=[100, 200], heads=3 * 2, kv=2), dict(qlens=[1, 30], lens=[100, 31], heads=5, kv=1),
                                           dict(qlens=[2, 61], lens=[100, 61], heads=14, kv=2)],
    "a few drafted tokens": dict(qlens=[4, 1, 5, 2], lens=[900, 44, 5, 1030], heads=16, kv=4, kind="bf16", bs=64),
    "sequences without tokens, without positions": dict(qlens=[0, 2, 0, 0, 1, 0], lens=[50, 20, 0, 0, 1, 3000], heads=4, kv=2),
    "no tokens at all": [dict(qlens=[0, 0], lens=[70, 0], heads=4, kv=2, pad=5), dict(qlens=[0, 0], lens=[70, 64], heads=4, kv=2, pad=5, shared=64),
                         dict(qlens=[0] * 9, lens=[70] * 9, heads=4, kv=2, pad=50, shared=64, max_q=50)],
    "starts past the tokens": [dict(qlens=[3, 6], lens=[30, 60], heads=4, kv=1, cut=5), dict(qlens=[30, 60], lens=[30, 60], heads=4, kv=1, cut=50),
                               dict(qlens=[30, 60], lens=[300, 330], heads=4, kv=1, cut=50, shared=256)],
    "prompts": dict(qlens=[33, 129, 1, 64, 65], lens=[33, 129, 1, 64, 65], heads=8, kv=2),
    "a prompt, heads of 64": dict(qlens=[300], lens=[300], heads=4, kv=4, dim=64, kind="bf16", bs=64),
    "chunks after cached positions": dict(qlens=[100, 17, 40], lens=[612, 17, 1025], heads=4, kv=1, kind="bf16", bs=128),
    "blocks of 1024": dict(qlens=[1, 50], lens=[1500, 1100], heads=4, kv=2, bs=1024, width_more=0),
    "prompts and single tokens together": dict(qlens=[1, 200, 1, 1, 3], lens=[900, 200, 2, 64, 333], heads=8, kv=2, pad=21),
    "cap": dict(qlens=[1, 70, 3], lens=[500, 90, 3], heads=8, kv=2, cap=3.0, spread=2.0),
    "cap, bf16": dict(qlens=[1, 70, 3], lens=[500, 90, 3], heads=8, kv=2, cap=30.0, spread=4.0, kind="bf16"),
    "distance bias": dict(qlens=[1, 70, 3], lens=[3000, 90, 700], heads=8, kv=2, alibi=True, kind="bf16"),
    "distance bias, cap, window": dict(qlens=[1, 130, 3], lens=[3000, 190, 700], heads=8, kv=2, alibi=True, cap=20.0, window=100),
    "window of one": dict(qlens=[1, 70, 2], lens=[500, 70, 90], heads=4, kv=1, window=1),
    "window of 512": dict(qlens=[1, 600, 2], lens=[2000, 700, 513], heads=4, kv=1, window=512, kind="bf16"),
    "documents": dict(qlens=[250, 1, 40], lens=[250, 300, 500], heads=4, kv=1, lo=lambda p: p // 37 * 37),
    "documents, distance bias, heads of 64": dict(qlens=[250, 1], lens=[250, 300], heads=4, kv=2, dim=64, lo=lambda p: p // 100 * 100, alibi=True, kind="bf16"),
    "prefix mask": dict(qlens=[250, 1, 40], lens=[250, 300, 90], heads=4, kv=2, hi=lambda p: np.maximum(p + 1, 120)),
    "prefix mask, distance bias, window": dict(qlens=[250, 40], lens=[250, 90], heads=4, kv=2, hi=lambda p: np.maximum(p + 1, 70), alibi=True, window=30, dim=64),
    "limits beyond the sequence": dict(qlens=[50, 1], lens=[60, 10], heads=4, kv=1, lo=lambda p: p * 0 - 9, hi=lambda p: p * 0 + 2 ** 31 - 1),
    "rows that see nothing": dict(qlens=[90, 1, 1, 5], lens=[150, 30, 31, 900], heads=4, kv=1, lo=lambda p: np.where(p % 3 == 0, p + 1, 0), kind="bf16"),
    "nothing seen at all": dict(qlens=[40, 1], lens=[50, 500], heads=4, kv=1, hi=lambda p: p * 0),
    "bounds shorter than the sequences": dict(qlens=[40, 1, 3], lens=[200, 500, 90], heads=4, kv=1, max_q=7, max_len=160),
    "bounds shorter than the sequences, window": [dict(qlens=[9, 3], lens=[300, 200], heads=4, kv=1, max_q=2, window=40),
                                                  dict(qlens=[9, 3], lens=[300, 200], heads=4, kv=1, max_q=2, window=40, hi=lambda p: p + 100)],
    "bounds of zero": [dict(qlens=[3, 1], lens=[30, 19], heads=4, kv=1, **kw) for kw in (dict(max_q=0), dict(max_q=0, shared=16), dict(max_len=0))] +
                      [dict(qlens=[90, 1], lens=[300, 219], heads=4, kv=1, **kw) for kw in (dict(max_q=0, shared=208), dict(max_len=0))],
    "loose bounds": dict(qlens=[1, 2], lens=[200, 90], heads=16, kv=4, max_q=900, width_more=300, max_len=4000),
    "no lse": dict(qlens=[1, 30, 2], lens=[700, 90, 3], heads=4, kv=1, with_lse=False),
    "token-major cache": dict(qlens=[1, 100, 3], lens=[700, 100, 90], heads=8, kv=4, token_major=True, kind="bf16"),
    "lost blocks": dict(qlens=[1, 100, 3, 1], lens=[700, 300, 90, 10], heads=8, kv=2, lost=[(0, 3), (0, 43), (1, 0), (1, 18), (2, 5), (3, 0)]),
    "values that are not finite": [dict(qlens=[100, 1, 1], lens=[300, 129, 90], heads=4, kv=2, poison=poison(*ODD), kind=k, dim=d) for k, d in (("f16", 128), ("bf16", 64))],
    "values that are not finite, window, mask": [dict(qlens=[100, 1, 4], lens=[300, 129, 90], heads=4, kv=1, poison=poison(*ODD), window=60),
                                                 dict(qlens=[100, 1, 4], lens=[300, 129, 90], heads=4, kv=1, poison=poison(*ODD), lo=lambda p: p // 50 * 50, kind="bf16"),
                                                 dict(qlens=[100, 1, 4], lens=[300, 129, 90], heads=4, kv=1, poison=poison(*ODD), hi=lambda p: np.minimum(p + 1, 128), kind="bf16")],
    "values that are not finite, shared prefix": [dict(qlens=[1, 2, 1], lens=[300, 290, 270], shared=256, heads=h, kv=1, lo=lambda p: p % 3 * 50 + 180, poison=poison(
        (0, 250, "v", INF, SOME), (0, 251, "v", NAN, slice(60, 62)), (0, 20, "v", -INF, SOME), (0, 200, "v", INF, slice(0, 1)), (1, 289, "v", NAN, slice(9, 10)))) for h in (4, 16)],
    "keys that are not finite": [dict(qlens=[100, 1, 3], lens=[300, 129, 90], heads=4, kv=1, kind="bf16", poison=poison((0, 270, "k", NAN, SOME), (1, 128, "k", INF, slice(0, 1)),
                                                                                                            (2, 88, "k", INF, SOME)))],
    "shared prefix, one token each": dict(qlens=[1] * 7, lens=[512 + 1 + 13 * s for s in range(7)], shared=512, heads=16, kv=4),
    "shared prefix, bf16, many": dict(qlens=[1] * 40, lens=[1024 + 1 + (29 * s) % 200 for s in range(40)], shared=1024, heads=8, kv=2, kind="bf16", bs=64),
    "shared prefix, heads of 64, drafts": dict(qlens=[1, 4, 3, 0, 2], lens=[300, 330, 291, 288, 500], shared=288, heads=6, kv=2, dim=64, bs=32),
    "shared prefix is everything but the token": dict(qlens=[1, 1, 1], lens=[65, 65, 65], shared=64, heads=4, kv=1),
    "shared prefix, window inside and outside": [dict(qlens=[1, 2, 1], lens=[600, 530, 900], shared=512, heads=4, kv=1, window=w) for w in (50, 300, 700)],
    "shared prefix, cap, distance bias": dict(qlens=[1, 2, 1], lens=[600, 530, 900], shared=512, heads=8, kv=2, cap=9.0, alibi=True, kind="bf16"),
    "shared prefix, prompts": dict(qlens=[100, 1, 300], lens=[356, 300, 556], shared=256, heads=8, kv=2, pad=9),
    "shared prefix, limits": dict(qlens=[20, 1, 3], lens=[300, 280, 290], shared=256, heads=4, kv=1, lo=lambda p: p // 100 * 100, hi=lambda p: np.maximum(p + 1, 262)),
    "shared prefix longer than a sequence": dict(qlens=[1, 2, 5], lens=[100, 300, 129], shared=256, heads=4, kv=1, max_len=300),
    "heads of 64, tiles that end inside": [dict(qlens=[60, 1, 90], lens=[300, 260, 90 + 144], heads=6, kv=2, dim=64, shared=144, kind=k, pad=3) for k in ("f16", "bf16")],
    "heads of 64, lost blocks and values that are not finite": [
        dict(qlens=[100, 1, 40], lens=[300, 129, 700], heads=4, kv=1, dim=64, lost=[(0, 2), (0, 17), (2, 8), (2, 43)], poison=poison(*ODD), window=w) for w in (0, 90)],
    "heads of 64, far positions": dict(qlens=[70, 2], lens=[2300, 1111], heads=4, kv=1, dim=64, cap=20.0, alibi=True, bs=128),
    "a prompt beside positions of one chunk and of more": [dict(qlens=[40, 1, 2], lens=[100, n, n - 5], heads=8, kv=2, window=w) for n, w in ((2047, 0), (2049, 0), (2100, 2017), (2100, 2018))],
    "a batch over shared positions, in chunks and in tiles": [dict(qlens=[1] * n, lens=[1200 + 16 * (s % 3) for s in range(n)], heads=4, kv=1, shared=1184, kind=k) for n, k in
                                                                     ((32, "f16"), (255, "bf16"), (257, "f16"))],
    "runs, windows": [dict(qlens=[150, 3], lens=[n, n], heads=4, kv=1, window=w) for n, w in ((383, 0), (385, 0), (1300, 351), (1300, 353), (1300, 900))],
    "shared prefix, lost blocks": dict(qlens=[1, 2], lens=[300, 290], shared=256, heads=4, kv=2, lost=[(0, 5), (1, 5), (1, 17)]),
}


@pytest.mark.parametrize("name", list(ATTN))
def test_attention(name):
    cases = ATTN[name] if isinstance(ATTN[name], list) else [ATTN[name]]
    for i, c in enumerate(cases):
        b = Batch(np.random.default_rng(sum(map(ord, name)) + i), **c)
        print(f"\n  {name} {i}: q {b.qlens[:8]} len {b.lens[:8]}", flush=True)
        with Dev() as d:
            a = b.upload(d)
            M.check(d.lib.mmoe_attn_paged(a, b.cache), "attention")
            b.check(d, name)


@pytest.mark.parametrize("qlen,shared,kind", [(1, 0, "f16"), (40, 0, "f16"), (3, 16384, "f16"), (40, 16384, "f16"), (40, 0, "bf16")])
def test_a_tail_of_small_weights(qlen, shared, kind):
    """one position with all the weight and no value, 20000 with some 2^-24.2 of it each and values: the result is the tail's"""
    rng = np.random.default_rng(21)
    b = Batch(rng, qlens=[qlen, 1], lens=[20000, 16500], shared=shared, heads=2, kv=1, dim=64, bs=128, kind=kind)
    k, v, q = (np.zeros(x.shape) for x in (b.k, b.v, b.q))
    q[..., 0] = 8.0
    k[..., 0] = 0.25 + 2.0 ** -6 * rng.integers(-4, 5, k.shape[:-1])
    v[:] = rng.uniform(90, 110, v.shape)
    for s, p in ((0, 777), (1, 9)):
        k[b.table[s, p // 128], p % 128, :, 0] = 17.0
        v[b.table[s, p // 128], p % 128] = 0
    b.k, b.v, b.q = (encode(x, kind) for x in (k, v, q))
    with Dev() as d:
        a = b.upload(d)
        M.check(d.lib.mmoe_attn_paged(a, b.cache), "attention")
        b.check(d, f"tail, {qlen} tokens, {shared} shared")


def test_attention_of_most_sequences():
    rng = np.random.default_rng(4)
    for shared in (0, 32):
        b = Batch(rng, qlens=[1] * M.KV_MAXSEQ, lens=[shared + 1 + s % 3 for s in range(M.KV_MAXSEQ)], shared=shared, heads=2, kv=1, dim=64)
        with Dev() as d:
            a = b.upload(d)
            M.check(d.lib.mmoe_attn_paged(a, b.cache), "attention")
            b.check(d, f"4096 sequences, {shared} shared")


def test_offsets_past_32_bits():
    """a cache whose blocks lie 2^25 values apart: the last one begins at byte 8.6e9"""
    rng = np.random.default_rng(8)
    n, bs, dim, kv, heads, apart = 129, 16, 64, 1, 4, 1 << 25
    lens, qlens = [2000, 40], [1, 30]
    b = Batch(rng, qlens=qlens, lens=lens, heads=heads, kv=kv, dim=dim, bs=bs, kind="bf16")
    assert b.nblocks > 128
    with Dev() as d:
        a = b.upload(d)
        c = b.cache
        c.block_stride = apart
        c.k = d.room((b.nblocks - 1) * apart * 2 + bs * dim * 2 + 4096)
        c.v = c.k + bs * dim * 2
        for i in range(b.nblocks):
            d.write(c.k + i * apart * 2, b.k[i].transpose(1, 0, 2))
            d.write(c.v + i * apart * 2, b.v[i].transpose(1, 0, 2))
        M.check(d.lib.mmoe_attn_paged(a, c), "attention")
        b.check(d, "far blocks")
        # and the write of keys and values
        x = encode(rng.standard_normal((3, 3 * dim)), "bf16")
        slot = np.array([(b.nblocks - 1) * bs + 3, 5, (b.nblocks - 2) * bs], np.int32)
        px = d.put(x)
        r = M.Rope(q=px, k=px + dim * 2, v=px + 2 * dim * 2, q_out=d.room(4096), q_token=3 * dim, q_head=dim, k_token=3 * dim, k_head=dim, v_token=3 * dim, v_head=dim,
                   qo_token=dim, qo_head=dim, pos=d.put(np.zeros(3, np.int32)), slot=d.put(slot), freq=d.put(np.ones(dim // 2)), ntok=3, heads=1, kv_heads=1,
                   head_dim=dim, rot=dim, in_dtype=M.BF16, out_dtype=M.BF16, mag=1.0)
        M.check(d.lib.mmoe_rope_kv(r, c), "rope")
        for t, s in enumerate(slot.tolist()):   # position 0: the rotation changes nothing
            row = d.get(c.v + (s // bs * apart + s % bs * dim) * 2, np.zeros(dim, np.uint16))
            assert np.array_equal(row, x[t, 2 * dim:])
            row = d.get(c.k + (s // bs * apart + s % bs * dim) * 2, np.zeros(dim, np.uint16))
            assert np.array_equal(row, x[t, dim:2 * dim])


class Server:
    """Sequences that come and go over one layer's blocks: the three operators together, step by step, and what they should hold"""
    H, KV, D, BS, ROT, N, WIDTH, NB = 8, 2, 128, 16, 64, 6, 24, 80

    def __init__(self, d, rng, ntok):
        self.d, self.rng, self.ntok, h, kv, dim = d, rng, ntok, self.H, self.KV, self.D
        freq = np.zeros(self.ROT // 2)
        M.check(d.lib.mmoe_rope_freqs(self.ROT, 10000.0, 1.0, 0, 0.0, 0.0, M.ptr(freq)), "freqs")
        self.freq, n, w = freq, self.N, self.WIDTH
        self.seen = [[] for _ in range(n)]       # (key, value) of each cached position, as the cache holds them
        z = lambda *s: np.zeros(s, np.int32)  # noqa: E731
        self.len, self.add, self.done, self.table = d.put(z(n)), d.put(z(n)), d.put(z(n)), d.put(z(n, w) - 1)
        self.free, self.nfree = d.put(np.arange(self.NB, dtype=np.int32)), d.put(np.array([self.NB], np.int32))
        self.qstart, self.pos, self.slot = d.put(z(n + 1)), d.put(z(ntok)), d.put(z(ntok))
        self.row = (h + 2 * kv) * dim
        self.x, self.q, self.out = d.room(ntok * self.row * 4), d.room(ntok * h * dim * 2), d.room(ntok * h * dim * 2)
        shape = (self.NB, kv, self.BS, dim)
        self.kc, self.vc, self.shape = d.put(encode(np.full(shape, np.nan), "f16")), d.put(encode(np.full(shape, np.nan), "f16")), shape
        self.cache = M.KvCache(k=self.kc, v=self.vc, block_stride=kv * self.BS * dim, head_stride=self.BS * dim, token_stride=dim, nblocks=self.NB, block_size=self.BS,
                               heads=kv, head_dim=dim, dtype=M.F16)
        self.plan = M.KvPlan(ctx=self.len, add=self.add, done=self.done, table=self.table, free_list=self.free, nfree=self.nfree, nfree_out=self.nfree, len=self.len,
                             qstart=self.qstart, pos=self.pos, slot=self.slot, nseq=n, width=w, nblocks=self.NB, block_size=self.BS, ntok=ntok)
        self.rope = M.Rope(q=self.x, k=self.x + h * dim * 4, v=self.x + (h + kv) * dim * 4, q_out=self.q, q_token=self.row, q_head=dim, k_token=self.row, k_head=dim,
                           v_token=self.row, v_head=dim, qo_token=h * dim, qo_head=dim, pos=self.pos, slot=self.slot, freq=d.put(freq), ntok=ntok, heads=h, kv_heads=kv,
                           head_dim=dim, rot=self.ROT, in_dtype=M.F32, out_dtype=M.F16, mag=1.0)
        self.attn = M.PagedAttn(q=self.q, out=self.out, q_token=h * dim, q_head=dim, out_token=h * dim, out_head=dim, qstart=self.qstart, len=self.len, table=self.table,
                                nseq=n, ntok=ntok, heads=h, width=w, max_q=ntok, max_len=w * self.BS, scale=dim ** -0.5)
        size = d.lib.mmoe_attn_paged_ws(self.attn, self.cache)
        self.attn.ws, self.attn.ws_bytes = d.room(size), size

    def queue(self):
        lib = self.d.lib
        M.check(lib.mmoe_kv_plan(self.plan), "plan")
        M.check(lib.mmoe_rope_kv(self.rope, self.cache), "rope")
        M.check(lib.mmoe_attn_paged(self.attn, self.cache), "attention")

    def feed(self, add, done):
        self.add_now, self.done_now = add, done
        self.x_now = self.rng.standard_normal((self.ntok, self.row)).astype(np.float32)
        self.d.write(self.add, np.array(add, np.int32)); self.d.write(self.done, np.array(done, np.int32)); self.d.write(self.x, self.x_now)

    def check(self, note):
        from paged_ref import attend
        d, h, kv, dim, n = self.d, self.H, self.KV, self.D, self.N
        table, start, length = d.get(self.table, np.zeros((n, self.WIDTH), np.int32)), d.get(self.qstart, np.zeros(n + 1, np.int32)), d.get(self.len, np.zeros(n, np.int32))
        kc, vc = (decode(d.get(p, np.zeros(self.shape, np.uint16)), "f16") for p in (self.kc, self.vc))
        out = decode(d.get(self.out, np.zeros((self.ntok, h, dim), np.uint16)), "f16")
        q = decode(d.get(self.q, np.zeros((self.ntok, h, dim), np.uint16)), "f16")
        x = self.x_now.reshape(self.ntok, h + 2 * kv, dim).astype(np.float64)
        used = []
        for s in range(n):
            if self.done_now[s]:
                self.seen[s] = []
            t = np.arange(start[s], start[s + 1])
            assert len(t) == self.add_now[s]
            p = len(self.seen[s]) + np.arange(len(t))
            want_k, want_q = rotate(x[t, h:h + kv], p, self.freq, self.ROT, 0, 1.0), rotate(x[t, :h], p, self.freq, self.ROT, 0, 1.0)
            assert (np.abs(q[t] - want_q) <= HALF["f16"] * np.abs(want_q) + 2.0 ** -19).all(), note
            self.seen[s] += [(a, b) for a, b in zip(want_k, x[t, h + kv:])]
            assert length[s] == len(self.seen[s]), (note, s)
            if not len(self.seen[s]):
                continue
            at = np.arange(length[s])
            blocks = table[s, at // self.BS]
            used += sorted(set(blocks.tolist()))
            k, v = kc[blocks, :, at % self.BS], vc[blocks, :, at % self.BS]
            wk, wv = np.array([a for a, _ in self.seen[s]]), np.array([b for _, b in self.seen[s]])
            assert (np.abs(k - wk) <= HALF["f16"] * np.abs(wk) + 2.0 ** -19).all() and (np.abs(v - wv) <= HALF["f16"] * np.abs(wv) + 2.0 ** -25).all(), (note, s)
            if len(t):
                o, _, off, _ = attend(q[t], k, v, p, at <= p[:, None], dim ** -0.5, 0.0, None, HALF["f16"])
                assert (np.abs(out[t] - o) <= off).all(), (note, s, np.abs(out[t] - o).max())
        assert len(used) == len(set(used)), "a block in two tables"
        assert d.get(self.nfree, np.zeros(1, np.int32))[0] == self.NB - len(used), note
        print(f"  {note}: lengths {length.tolist()}", flush=True)


def test_steps_of_a_server():
    """prompts, then single tokens, sequences that end and others that begin in their rows"""
    with Dev() as d:
        s = Server(d, np.random.default_rng(21), 260)
        for i, (add, done) in enumerate([([100, 7, 0, 33, 1, 0], [0] * 6), ([1, 1, 60, 1, 1, 0], [0] * 6), ([1, 1, 1, 1, 1, 140], [0] * 6), ([1, 0, 1, 40, 1, 1], [0, 1, 0, 1, 0, 0]),
                                         ([1, 90, 1, 1, 0, 1], [0] * 6), ([0] * 6, [1, 0, 0, 0, 1, 0]), ([150, 1, 1, 1, 1, 1], [0] * 6)]):
            s.feed(add, done)
            s.queue()
            s.check(f"step {i}")


def test_captured_step_replayed_with_others_between():
    """one step captured into a graph, replayed for growing, ending and new sequences, with eager steps of another server between"""
    with Dev() as d:
        s, other = Server(d, np.random.default_rng(5), 6), Server(d, np.random.default_rng(6), 200)
        s.feed([1, 1, 0, 1, 1, 1], [0] * 6)
        s.queue()
        s.check("eager")
        hip = C.CDLL("libamdhip64.so")
        stream, graph, ex = C.c_void_p(d.lib.mmoe_stream()), C.c_void_p(), C.c_void_p()
        assert hip.hipStreamBeginCapture(stream, 1) == 0
        s.queue()
        assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
        assert hip.hipGraphInstantiate(C.byref(ex), graph, None, None, C.c_size_t(0)) == 0
        try:
            for i in range(20):
                done = [1 if (i * 5 + j) % 11 == 0 else 0 for j in range(6)]
                s.feed([0 if (i + j) % 7 == 0 else 1 for j in range(6)], done)
                assert hip.hipGraphLaunch(ex, stream) == 0
                s.check(f"replay {i}")
                if i % 4 == 0:
                    other.feed([20, 0, 5, 1, 30, 1], [1, 1, 0, 1, 1, 0] if i else [0] * 6)
                    other.queue()
                    other.check(f"eager between, {i}")
        finally:
            hip.hipGraphExecDestroy(ex); hip.hipGraphDestroy(graph)


def test_two_calls_at_once_with_workspaces_of_their_own():
    """two captured attention calls replayed on two other streams at the same time"""
    rng = np.random.default_rng(31)
    bs = [Batch(rng, qlens=[1] * 5, lens=[900 + 100 * i for i in range(5)], heads=8, kv=2), Batch(rng, qlens=[1, 3, 60], lens=[700, 800, 900], shared=512, heads=8, kv=2, kind="bf16")]
    hip = C.CDLL("libamdhip64.so")
    with Dev() as d:
        made = []
        for b in bs:
            a = b.upload(d)
            lib_stream, graph, ex, st = C.c_void_p(d.lib.mmoe_stream()), C.c_void_p(), C.c_void_p(), C.c_void_p()
            assert hip.hipStreamBeginCapture(lib_stream, 1) == 0
            M.check(d.lib.mmoe_attn_paged(a, b.cache), "attention")
            assert hip.hipStreamEndCapture(lib_stream, C.byref(graph)) == 0
            assert hip.hipGraphInstantiate(C.byref(ex), graph, None, None, C.c_size_t(0)) == 0
            assert hip.hipStreamCreate(C.byref(st)) == 0
            made.append((graph, ex, st))
        try:
            assert hip.hipDeviceSynchronize() == 0
            for i in range(30):
                for _, ex, st in made:
                    assert hip.hipGraphLaunch(ex, st) == 0
            assert hip.hipDeviceSynchronize() == 0
            for b in bs:
                b.check(d, "two at once")
        finally:
            for graph, ex, st in made:
                hip.hipGraphExecDestroy(ex); hip.hipGraphDestroy(graph); hip.hipStreamDestroy(st)


def test_results_repeat_and_do_not_depend_on_the_workspace():
    rng = np.random.default_rng(77)
    for kw in (dict(qlens=[1, 2, 70], lens=[5000, 600, 700], heads=8, kv=2), dict(qlens=[1] * 9, lens=[1500 + s for s in range(9)], shared=1024, heads=16, kv=4, kind="bf16")):
        b = Batch(rng, **kw)
        with Dev() as d:
            a = b.upload(d)
            got = []
            for fill in (0, 0xff, 0x7f):
                d.write(a.ws, np.full(a.ws_bytes, fill, np.uint8))
                M.check(d.lib.mmoe_attn_paged(a, b.cache), "attention")
                got.append(d.get(b.p_out, b.out0))
            assert all(np.array_equal(g, got[0]) for g in got[1:])
            b.check(d, "workspace of any content")
            a.ws_bytes -= 1
            assert d.lib.mmoe_attn_paged(a, b.cache) == -1 and b"workspace" in d.lib.mmoe_last_error()
            a.ws_bytes += 1


def test_profile_counts_the_operators():
    rng = np.random.default_rng(1)
    b = Batch(rng, qlens=[1], lens=[100], heads=4, kv=1)
    with Dev() as d:
        a = b.upload(d)
        ms, cnt = C.c_double(), C.c_long()
        M.check(d.lib.mmoe_prof_reset(), "reset"); M.check(d.lib.mmoe_prof(1), "prof")
        try:
            M.check(d.lib.mmoe_attn_paged(a, b.cache), "attention")
        finally:
            M.check(d.lib.mmoe_prof(0), "prof off")
        M.check(d.lib.mmoe_prof_get(M.KERNELS.index("att_paged"), C.byref(ms), C.byref(cnt)), "get")
        assert cnt.value == 1 and 0 < ms.value < 50
        b.check(d, "profiled")
