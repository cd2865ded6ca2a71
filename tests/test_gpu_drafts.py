"""Drafted tokens (include/maplemoe.h, Part 3) on the card, against plain numpy in 64 bits."""
import ctypes as C

import numpy as np
import pytest

import maplemoe as M
from draft_ref import TreeBatch, accept, paths, tree, tree_plan
from paged_ref import HALF, Dev, attend, decode, encode, rotate

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------------- what drafted tokens follow
def run_tree_plan(qstart, length, parent, words, ntok):
    with Dev() as d:
        pos, bits = np.full(ntok, -9, np.int32), np.full((ntok, words), 5, np.uint64)
        p_pos, p_bits = d.put(pos), d.put(bits)
        a = M.TreePlan(qstart=d.put(np.array(qstart, np.int32)), len=d.put(np.array(length, np.int32)), parent=d.put(np.array(parent, np.int32)), pos=p_pos, bits=p_bits,
                       nseq=len(length), ntok=ntok, words=words)
        M.check(d.lib.mmoe_tree_plan(a), "mmoe_tree_plan")
        return d.get(p_pos, pos), d.get(p_bits, bits)


@pytest.mark.parametrize("sizes,back,words,pad", [([1], 1, 1, 0), ([64, 0, 63, 1, 33], 12, 1, 5), ([65, 128, 7], 3, 2, 0), ([192, 130], 1, 3, 300), ([512, 511, 257, 40], 9, 8, 1),
                                                  ([512], 1, 8, 0), ([300], 400, 5, 0), ([70, 64, 3], 5, 1, 2), ([600, 20], 4, 8, 0), ([4] * 4096, 3, 1, 9)])
def test_tree_plan(sizes, back, words, pad):
    """nodes past the words, and trees past MMOE_TREE_MAX, among them"""
    print(f"\n  {sizes[:6]} back={back} words={words}", flush=True)
    rng = np.random.default_rng(len(sizes) + back)
    qstart = np.concatenate([[0], np.cumsum(sizes)])
    parent = np.concatenate([tree(rng, n, back) for n in sizes] + [np.full(pad, 3)]).astype(np.int64)
    length = qstart[1:] - qstart[:-1] + rng.integers(0, 1 << 29, len(sizes))
    got, want = run_tree_plan(qstart, length, parent, words, len(parent)), tree_plan(qstart, length, parent, words, len(parent))
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_tree_plan_of_forests_and_of_parents_that_are_none():
    parent = [-1, -1, 0, 1, -1, 4, 5, 99, 8, -7, 2 ** 31 - 1, -2 ** 31, 10]   # itself, later ones, none of the tree: followers of nobody
    got, want = run_tree_plan([0, 13], [20], parent, 1, 13), tree_plan([0, 13], [20], parent, 1, 13)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    pos, bits = run_tree_plan([0], [], [3] * 500, 2, 500)       # a batch without sequences: room for tokens only
    assert not pos.any() and not bits.any()


# ---------------------------------------------------------------------------------------------------- attention
def drafts(rng, sizes, back):
    return [paths(tree(rng, n, back)) for n in sizes]


CASES = [  # nodes, cached positions, back, options
    ([1], [0], 1, dict()),
    ([1], [77], 1, dict(kind="bf16")),
    ([4], [30], 2, dict(heads=8, kv=2)),
    ([3, 1, 4], [100, 0, 517], 2, dict(heads=8, kv=2, kind="bf16", pad=3)),
    ([16], [40], 5, dict(heads=4, kv=4, dim=64)),
    ([17], [47], 5, dict(heads=4, kv=4, dim=64, kind="bf16")),
    ([26], [700], 12, dict(heads=16, kv=4)),
    ([33, 64, 2, 11], [65, 190, 1300, 0], 12, dict(heads=8, kv=2, kind="bf16", pad=2)),
    ([33, 64, 2, 11], [64, 127, 1000, 3], 1, dict(heads=8, kv=2, token_major=True, bs=64)),
    ([61, 9], [400, 33], 60, dict(heads=6, kv=2, dim=64, bs=32)),
    ([64, 64], [100, 200], 12, dict(heads=2, kv=1, window=32)),
    ([64, 30, 5], [100, 200, 900], 2, dict(heads=2, kv=1, window=7, kind="bf16")),
    ([4, 2], [1000, 90], 2, dict(heads=4, kv=1, window=50)),
    ([40, 3], [300, 120], 6, dict(heads=4, kv=2, cap=20.0, kind="bf16")),
    ([40, 3], [300, 120], 6, dict(heads=4, kv=2, alibi=True)),
    ([4], [300], 2, dict(heads=4, kv=1, alibi=True, kind="bf16")),
    ([4, 3], [30, 5], 1, dict(heads=4, kv=1, alibi=True, cap=30.0)),
    ([61, 20], [70, 190], 12, dict(heads=12, kv=12, dim=64, alibi=True, cap=15.0, window=100)),
    ([61, 64, 5], [130, 64 + 70, 200], 1, dict(heads=4, kv=4, dim=64, alibi=True, shared=64, kind="bf16")),
    ([9, 30, 1, 2], [260, 300, 256, 999], 4, dict(heads=8, kv=2, shared=256, kind="bf16")),
    ([2, 3, 1], [70, 64, 90], 2, dict(heads=4, kv=2, shared=64)),
    ([100], [90], 9, dict(heads=4, kv=2)),
    ([200, 65, 129], [10, 500, 0], 5, dict(heads=2, kv=1, kind="bf16", words=4)),
    ([130, 70], [33, 200], 40, dict(heads=2, kv=2, dim=64, alibi=True, words=3)),
    ([130, 140], [600, 128], 1, dict(heads=2, kv=1, window=90, alibi=True, words=3, kind="bf16")),
    ([512], [100], 9, dict(heads=1, kv=1, dim=64, words=8)),
    ([5], [30], 2, dict(heads=4, kv=1, words=8)),
    ([20, 40], [5000, 2000], 6, dict(heads=4, kv=1)),
    ([3], [9000], 2, dict(heads=4, kv=1, kind="bf16")),
]


@pytest.mark.parametrize("i", range(len(CASES)))
def test_attention_of_drafts(i):
    sizes, ctx, back, kw = CASES[i]
    print(f"\n  {sizes} over {ctx}, {kw}", flush=True)
    rng = np.random.default_rng(100 + i)
    b = TreeBatch(rng, drafts(rng, sizes, back), lens=[c + n for c, n in zip(ctx, sizes)], **kw)
    with Dev() as d:
        b.run(d, f"case {i}")


@pytest.mark.parametrize("alibi", [False, True])
@pytest.mark.parametrize("n,ctx,heads,kv,dim", [(3, 5, 4, 1, 128), (40, 100, 4, 2, 128), (70, 31, 4, 4, 64), (64, 0, 2, 1, 64)])
def test_any_bits(n, ctx, heads, kv, dim, alibi):
    """bits that are no tree's: any earlier tokens, none at all, the token itself left out, and ones past it, which count for nothing"""
    rng = np.random.default_rng(n)
    rows = rng.random((n, n)) < 0.3
    rows[1] = False
    rows[n - 1] = True
    b = TreeBatch(rng, [rows, rng.random((n, n)) < 0.8], lens=[ctx + n, ctx + n + 300], heads=heads, kv=kv, dim=dim, alibi=alibi, kind="bf16")
    with Dev() as d:
        b.run(d, f"{n} tokens")
        if not ctx:
            out = decode(d.get(b.p_out, b.out0)[1, 8:8 + heads * (dim + 8)].reshape(heads, dim + 8)[:, :dim].copy(), "bf16")
            assert not out.any() and (d.get(b.p_lse, b.lse0)[1] == -np.inf).all()


@pytest.mark.parametrize("n,ctx,heads,dim", [(4, 200, 4, 128), (40, 90, 4, 64), (64, 1000, 4, 128)])
@pytest.mark.parametrize("what", ["nan", "inf", "seen"])
def test_values_of_other_paths_never_arrive(n, ctx, heads, dim, what):
    """keys and values of drafted tokens on other paths are NaN or infinite; with `seen` one that some tokens see is infinite"""
    print(f"\n  {n} {what}", flush=True)
    rng = np.random.default_rng(n + ctx)
    rows = paths(tree(rng, n, 3))
    hidden = [j for j in range(n) if not rows[n - 1, j]]
    rows = [rows[n - 1] & (np.arange(n) <= i) for i in range(n)]      # every token on the last one's path, as far as it is there
    rows[n - 1][hidden] = False

    def poison(b):
        for j in hidden:
            at, p = b.table[0, (ctx + j) // b.bs], (ctx + j) % b.bs
            if what == "nan":
                b.k[at, p] = b.v[at, p] = encode(np.full(dim, np.nan), b.kind)
            else:
                b.v[at, p] = encode(np.full(dim, np.inf), b.kind)
                b.k[at, p] = encode(np.full(dim, np.nan), b.kind)
        if what == "seen":
            j = [j for j in range(n) if rows[n - 1][j]][-2]
            b.v[b.table[0, (ctx + j) // b.bs], (ctx + j) % b.bs, 0, 3] = encode(np.array([-np.inf]), b.kind)[0]

    b = TreeBatch(rng, [np.array(rows)], lens=[ctx + n], heads=heads, kv=1, dim=dim, poison=poison)
    with Dev() as d:
        b.run(d, what)


def test_limits_of_documents_bounds_and_lost_blocks():
    rng = np.random.default_rng(3)
    sizes, ctx = [40, 3, 64], [300, 200, 500]
    lens = [c + n for c, n in zip(ctx, sizes)]
    rows = drafts(rng, sizes, 6)
    for kw in (dict(lo=lambda pos: 90 + (pos % 7) * 30), dict(lo=lambda pos: np.full(len(pos), 1 << 29)), dict(max_q=30), dict(max_q=2), dict(max_len=250), dict(max_len=310),
               dict(lost=[(0, 3), (0, 20), (1, 12), (2, 0), (2, 33)]), dict(cut=50, pad=7), dict(with_lse=False), dict(lo=lambda pos: pos - 100, window=64, alibi=True)):
        print(f"  {list(kw)}", flush=True)
        b = TreeBatch(rng, rows, lens=lens, heads=4, kv=2, kind="bf16", **kw)
        with Dev() as d:
            b.run(d, str(list(kw)))


def test_a_chain_is_plain_attention():
    """a draft without branches sees what mmoe_attn_paged's causal tokens see"""
    rng = np.random.default_rng(9)
    for sizes, ctx, kw in (([3, 4], [100, 900], dict(heads=4, kv=1)), ([30, 64, 7], [700, 64, 2000], dict(heads=8, kv=2, kind="bf16")), ([64, 20], [300, 260], dict(heads=4, kv=4, dim=64, shared=256, alibi=True))):
        b = TreeBatch(rng, drafts(rng, sizes, 1), lens=[c + n for c, n in zip(ctx, sizes)], **kw)
        with Dev() as d:
            b.run(d, "as a tree")
            d.write(b.p_out, b.out0); d.write(b.p_lse, b.lse0)
            a = b.args
            (a.ws, a.ws_bytes), tree_ws = b.plain_ws, (a.ws, a.ws_bytes)
            M.check(d.lib.mmoe_attn_paged(a, b.cache), "plain")
            b.check(d, "plain")
            a.ws, a.ws_bytes = tree_ws


def test_drafts_of_many_sequences():
    rng = np.random.default_rng(4)
    b = TreeBatch(rng, drafts(rng, [1 + s % 3 for s in range(M.KV_MAXSEQ)], 2), lens=[5 + s % 40 for s in range(M.KV_MAXSEQ)], heads=2, kv=1, dim=64)
    with Dev() as d:
        b.run(d, "4096 sequences")
    b = TreeBatch(rng, drafts(rng, [1 + s % 23 for s in range(70)], 5), lens=[25 + 9 * s for s in range(70)], heads=4, kv=1, kind="bf16")
    with Dev() as d:
        b.run(d, "70 sequences")


@pytest.mark.parametrize("shared", [0, 64])
def test_a_step_without_new_tokens(shared):
    """a captured step whose sequences all rest: the rows stay as they were, whatever the workspace holds of the step before"""
    rng = np.random.default_rng(5)
    b = TreeBatch(rng, drafts(rng, [9, 40], 5), lens=[900, 1500], heads=8, kv=2, shared=shared)
    with Dev() as d:
        b.run(d, "with tokens")
        d.write(b.p_out, b.out0); d.write(b.p_lse, b.lse0)
        d.write(b.args.qstart, np.zeros(3, np.int32))
        M.check(d.lib.mmoe_attn_tree(b.args, b.cache, b.p_bits, b.words), "attention")
        assert np.array_equal(d.get(b.p_out, b.out0), b.out0) and np.array_equal(d.get(b.p_lse, b.lse0), b.lse0)


@pytest.mark.parametrize("heads,kv,shared,most", [(8, 2, 0, 40), (4, 4, 64, 40), (64, 1, 0, 40)])
def test_starts_that_do_not_ascend(heads, kv, shared, most):
    """sequences that claim one another's tokens, in more row tiles than the tokens make: nothing is written outside the rows and the workspace"""
    rng = np.random.default_rng(heads)
    n = 60
    b = TreeBatch(rng, drafts(rng, [most] + [1] * (n - 1), 5), lens=[most + 200] + [200 + s for s in range(1, n)], heads=heads, kv=kv, shared=shared, pad=30)
    with Dev() as d:
        a = b.upload(d)
        last = b.ntok - 30
        for start in ([0, last] * (n // 2) + [last], [last] * n + [0], [0] + [last - 3 * s for s in range(n)], [0, 2 ** 31 - 1, -2 ** 31, last] * (n // 4) + [last]):
            d.write(a.qstart, np.array(start[:n + 1], np.int32))
            for fill in (0, 0x7f, 0xff):
                d.write(a.ws, np.full(a.ws_bytes, fill, np.uint8))
                M.check(d.lib.mmoe_attn_tree(a, b.cache, b.p_bits, b.words), "attention")
                raw = d.get(b.p_out, b.out0)
                body = raw[:, 8:8 + heads * 136].reshape(b.ntok, heads, 136)
                assert (raw[:, :8] == 0x1234).all() and (raw[:, 8 + heads * 136:] == 0x1234).all() and (body[:, :, 128:] == 0x1234).all()
                assert np.array_equal(d.get(a.ws + a.ws_bytes, b.ws_guard), b.ws_guard), "written behind the workspace"


def test_drafts_past_32_bits():
    """a cache whose blocks lie 2^25 values apart: the last one begins at byte 8.6e9"""
    rng = np.random.default_rng(8)
    bs, dim, kv, heads, apart = 16, 64, 1, 4, 1 << 25
    b = TreeBatch(rng, drafts(rng, [3, 30], 4), lens=[2003, 70], heads=heads, kv=kv, dim=dim, bs=bs, kind="bf16")
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
        M.check(d.lib.mmoe_attn_tree(a, c, b.p_bits, b.words), "attention")
        b.check(d, "far blocks")


def test_repeats_profile_and_other_stream():
    """the same bits from a workspace of any content; two captured calls replayed on two streams at once; the kernel ids count"""
    rng = np.random.default_rng(31)
    bs = [TreeBatch(rng, drafts(rng, [9, 40, 1], 5), lens=[900, 1500, 3000], heads=8, kv=2), TreeBatch(rng, drafts(rng, [2] * 7, 2), lens=[700 + 50 * i for i in range(7)], heads=8, kv=2, kind="bf16")]
    hip = C.CDLL("libamdhip64.so")
    with Dev() as d:
        made = []
        for b in bs:
            a = b.upload(d)
            got = []
            for fill in (0, 0xff):
                d.write(a.ws, np.full(a.ws_bytes, fill, np.uint8))
                M.check(d.lib.mmoe_attn_tree(a, b.cache, b.p_bits, b.words), "attention")
                got.append(d.get(b.p_out, b.out0))
            assert np.array_equal(got[0], got[1])
            lib_stream, graph, ex, st = C.c_void_p(d.lib.mmoe_stream()), C.c_void_p(), C.c_void_p(), C.c_void_p()
            assert hip.hipStreamBeginCapture(lib_stream, 1) == 0
            M.check(d.lib.mmoe_attn_tree(a, b.cache, b.p_bits, b.words), "attention")
            assert hip.hipStreamEndCapture(lib_stream, C.byref(graph)) == 0
            assert hip.hipGraphInstantiate(C.byref(ex), graph, None, None, C.c_size_t(0)) == 0
            assert hip.hipStreamCreate(C.byref(st)) == 0
            made.append((graph, ex, st))
        try:
            assert hip.hipDeviceSynchronize() == 0
            for i in range(20):
                for _, ex, st in made:
                    assert hip.hipGraphLaunch(ex, st) == 0
            assert hip.hipDeviceSynchronize() == 0
            for b in bs:
                b.check(d, "two at once")
        finally:
            for graph, ex, st in made:
                hip.hipGraphExecDestroy(ex); hip.hipGraphDestroy(graph); hip.hipStreamDestroy(st)
        ms, cnt = C.c_double(), C.c_long()
        M.check(d.lib.mmoe_prof_reset(), "reset"); M.check(d.lib.mmoe_prof(1), "prof")
        try:
            M.check(d.lib.mmoe_attn_tree(bs[0].args, bs[0].cache, bs[0].p_bits, bs[0].words), "attention")
        finally:
            M.check(d.lib.mmoe_prof(0), "prof off")
        M.check(d.lib.mmoe_prof_get(M.KERNELS.index("att_tree"), C.byref(ms), C.byref(cnt)), "get")
        assert cnt.value >= 1 and 0 < ms.value < 50


# ---------------------------------------------------------------------------------------------------- which drafted tokens stay
def run_accept(qstart, length, parent, token, choice, in_place=False):
    with Dev() as d:
        n, ntok = len(length), len(parent)
        i = lambda v: np.array(v, np.int32)  # noqa: E731
        kept, z = np.full(ntok, -77, np.int32), np.full(n, -5, np.int32)
        p_len, p_kept, p = d.put(i(length)), d.put(kept), [d.put(z) for _ in range(3)]
        ctx = p_len if in_place else p[1]
        a = M.TreeAccept(qstart=d.put(i(qstart)), len=p_len, parent=d.put(i(parent)), token=d.put(i(token)), next=d.put(i(choice)), kept=p_kept, count=p[0], ctx=ctx, last=p[2],
                         nseq=n, ntok=ntok)
        M.check(d.lib.mmoe_tree_accept(a), "mmoe_tree_accept")
        return d.get(p_kept, kept), d.get(p[0], z), d.get(ctx, z), d.get(p[2], z)


@pytest.mark.parametrize("sizes,back,vocab,in_place", [([1], 1, 2, False), ([40, 0, 63, 1, 33], 12, 3, True), ([512, 600, 130], 1, 1, False), ([300, 64, 65], 200, 4, False),
                                                       ([7] * 4096, 3, 2, True), ([512], 512, 1, False)])
def test_accept(sizes, back, vocab, in_place):
    """few tokens to choose from, so that siblings are alike and long paths agree; trees past MMOE_TREE_MAX"""
    print(f"\n  {sizes[:6]} back={back} vocab={vocab}", flush=True)
    rng = np.random.default_rng(len(sizes) + back)
    qstart = np.concatenate([[0], np.cumsum(sizes)])
    parent = np.concatenate([tree(rng, n, back) for n in sizes] + [[]]).astype(np.int64)
    length = qstart[1:] - qstart[:-1] + rng.integers(0, 1 << 29, len(sizes))
    token, choice = rng.integers(0, vocab, len(parent)), rng.integers(0, vocab, len(parent))
    if vocab == 1:
        assert accept(qstart, length, parent, token, choice, np.full(len(parent), -77))[1].max() > 1
    want, got = accept(qstart, length, parent, token, choice, np.full(len(parent), -77)), run_accept(qstart, length, parent, token, choice, in_place)
    for w, g in zip(want, got):
        assert np.array_equal(w, g)


def test_accept_where_parents_are_none():
    parent, token = [-1, -1, 0, 99, 4, -9, 2], [1] * 7     # roots beside node 0, a later one, itself: never accepted
    want, got = accept([0, 7], [50], parent, token, token, np.full(7, -77)), run_accept([0, 7], [50], parent, token, token)
    assert want[0][:3].tolist() == [43, 45, 49]
    for w, g in zip(want, got):
        assert np.array_equal(w, g)


def test_tokens_past_the_arrays():
    """a last sequence of which only some tokens lie inside the arrays: their positions are those that mmoe_attn_tree takes them to have"""
    rng = np.random.default_rng(7)
    qstart, length, ntok = np.array([0, 20, 50]), np.array([70, 130]), 41
    parent = np.array(tree(rng, 20, 3) + tree(rng, 30, 3), np.int64)
    pos, bits = tree_plan(qstart, length, parent, 1, 50)
    got = run_tree_plan(qstart, length, parent[:ntok], 1, ntok)
    assert np.array_equal(got[0], pos[:ntok]) and np.array_equal(got[1], bits[:ntok]) and pos[20] == 100
    token = np.arange(50)                       # only what lies inside is ever the model's choice
    choice = np.concatenate([np.full(20, 99), np.where(np.arange(20, 50) + 1 < ntok, np.arange(21, 51), 99)])
    parent[20:] = np.arange(-1, 29)
    want, out = accept(qstart, length, parent, token, choice, np.full(50, -77)), run_accept(qstart, length, parent[:ntok], token[:ntok], choice[:ntok])
    assert want[1].tolist() == [1, 21] and np.array_equal(out[0], want[0][:ntok])
    for w, g in zip(want[1:], out[1:]):
        assert np.array_equal(w, g)


# ---------------------------------------------------------------------------------------------------- the operators together
class Drafting:
    """A server that drafts: sequences whose next tokens are trees, accepted by a model that is a table of what follows what. Two layers' caches;
    what a position holds is known from its token and its place, so that after each step the caches can be checked against the accepted texts."""
    H, KV, D, BS, N, WIDTH, NB, VOCAB, LAYERS = 8, 2, 128, 16, 5, 12, 40, 6, 2

    def __init__(self, d, rng, ntok):
        self.d, self.rng, self.ntok, h, kv, dim, n, w = d, rng, ntok, self.H, self.KV, self.D, self.N, self.WIDTH
        z = lambda *s: np.zeros(s, np.int32)  # noqa: E731
        self.text = [[] for _ in range(n)]
        self.after = rng.integers(0, self.VOCAB, self.VOCAB)
        self.rows = rng.standard_normal((self.VOCAB, (h + 2 * kv) * dim)).astype(np.float32)
        self.freq = np.zeros(dim // 2)
        M.check(d.lib.mmoe_rope_freqs(dim, 10000.0, 1.0, 0, 0.0, 0.0, M.ptr(self.freq)), "freqs")
        self.len, self.ctx, self.add, self.table = d.put(z(n)), d.put(z(n)), d.put(z(n)), d.put(z(n, w) - 1)
        self.free, self.nfree = d.put(np.arange(self.NB, dtype=np.int32)), d.put(np.array([self.NB], np.int32))
        self.qstart, self.slot, self.pos, self.bits = d.put(z(n + 1)), d.put(z(ntok)), d.put(z(ntok)), d.put(np.zeros(ntok, np.uint64))
        self.parent, self.token, self.next, self.kept, self.count, self.last = (d.put(z(ntok)) for _ in range(6))
        self.x, self.q, self.out = d.room(ntok * (h + 2 * kv) * dim * 4), d.room(ntok * h * dim * 2), d.put(z(ntok, h, dim // 2))
        self.shape = (self.NB, kv, self.BS, dim)
        self.caches = (M.KvCache * self.LAYERS)(*(
            M.KvCache(k=d.put(encode(np.full(self.shape, np.nan), "f16")), v=d.put(encode(np.full(self.shape, np.nan), "f16")), block_stride=kv * self.BS * dim,
                      head_stride=self.BS * dim, token_stride=dim, nblocks=self.NB, block_size=self.BS, heads=kv, head_dim=dim, dtype=M.F16) for _ in range(self.LAYERS)))
        row = (h + 2 * kv) * dim
        pages = dict(nseq=n, width=w, nblocks=self.NB, block_size=self.BS)
        self.plan = M.KvPlan(ctx=self.ctx, add=self.add, table=self.table, free_list=self.free, nfree=self.nfree, nfree_out=self.nfree, len=self.len, qstart=self.qstart,
                             pos=d.put(z(ntok)), slot=self.slot, ntok=ntok, **pages)
        self.tree = M.TreePlan(qstart=self.qstart, len=self.len, parent=self.parent, pos=self.pos, bits=self.bits, nseq=n, ntok=ntok, words=1)
        self.rope = M.Rope(q=self.x, k=self.x + h * dim * 4, v=self.x + (h + kv) * dim * 4, q_out=self.q, q_token=row, q_head=dim, k_token=row, k_head=dim, v_token=row,
                           v_head=dim, qo_token=h * dim, qo_head=dim, pos=self.pos, slot=self.slot, freq=d.put(self.freq), ntok=ntok, heads=h, kv_heads=kv, head_dim=dim,
                           rot=dim, in_dtype=M.F32, out_dtype=M.F16, mag=1.0)
        self.attn = M.PagedAttn(q=self.q, out=self.out, q_token=h * dim, q_head=dim, out_token=h * dim, out_head=dim, qstart=self.qstart, len=self.len, table=self.table,
                                nseq=n, ntok=ntok, heads=h, width=w, max_q=64, max_len=w * self.BS, scale=dim ** -0.5)
        size = d.lib.mmoe_attn_tree_ws(self.attn, self.caches[0], self.bits, 1)
        self.attn.ws, self.attn.ws_bytes = d.room(size), size
        self.acc = M.TreeAccept(qstart=self.qstart, len=self.len, parent=self.parent, token=self.token, next=self.next, kept=self.kept, count=self.count, ctx=self.ctx,
                                last=self.last, nseq=n, ntok=ntok)
        self.com = M.KvCompact(table=self.table, first=self.qstart, count=self.count, kept=self.kept, nseq=n, width=w, nkept=ntok)
        self.fre = M.KvFree(ctx=self.len, keep=self.ctx, len=self.ctx, table=self.table, free_list=self.free, nfree=self.nfree, nfree_out=self.nfree, **pages)

    def queue(self):
        lib = self.d.lib
        M.check(lib.mmoe_kv_plan(self.plan), "plan")
        M.check(lib.mmoe_tree_plan(self.tree), "tree")
        for c in self.caches:
            M.check(lib.mmoe_rope_kv(self.rope, c), "rope")
            M.check(lib.mmoe_attn_tree(self.attn, c, self.bits, 1), "attention")
        M.check(lib.mmoe_tree_accept(self.acc), "accept")
        M.check(lib.mmoe_kv_compact(self.com, self.caches, self.LAYERS), "compact")
        M.check(lib.mmoe_kv_free(self.fre), "free")

    def feed(self, sizes):
        """a draft for each sequence: a node's children are the model's choice behind it, often, and others"""
        self.sizes, self.trees, self.tokens = sizes, [], []
        for s, n in enumerate(sizes):
            p = tree(self.rng, n, 4)
            t = []
            for i in range(n):
                if i == 0:
                    t.append(int(self.after[self.text[s][-1]]) if self.text[s] else s % self.VOCAB)
                else:
                    t.append(int(self.after[t[p[i]]]) if self.rng.random() < 0.5 else int(self.rng.integers(0, self.VOCAB)))
            self.trees.append(p); self.tokens.append(t)
        flat = np.zeros(self.ntok, np.int32)
        tok = np.concatenate([np.array(t, np.int64) for t in self.tokens])
        self.flat = tok
        par = np.concatenate([np.array(p, np.int64) for p in self.trees])
        for where, v in ((self.add, np.array(sizes)), (self.parent, par), (self.token, tok), (self.next, self.after[tok])):
            a = flat[:len(v)].copy() if where == self.add else flat.copy()
            a[:len(v)] = v
            self.d.write(where, a.astype(np.int32))
        x = np.zeros((self.ntok, self.rows.shape[1]), np.float32)
        x[:len(tok)] = self.rows[tok]
        self.d.write(self.x, x)

    def held(self, token, pos):
        """the key and value heads of a token at a position"""
        x = self.rows[token].reshape(-1, self.D).astype(np.float64)[None]
        return rotate(x[:, self.H:self.H + self.KV], np.array([pos]), self.freq, self.D, 0, 1.0)[0], x[0, self.H + self.KV:]

    def check(self, note):
        d, n, h, kv, dim = self.d, self.N, self.H, self.KV, self.D
        start = np.concatenate([[0], np.cumsum(self.sizes)])
        out, q = (decode(d.get(p, np.zeros((self.ntok, h, dim), np.uint16)), "f16") for p in (self.out, self.q))
        table, ctx = d.get(self.table, np.zeros((n, self.WIDTH), np.int32)), d.get(self.ctx, np.zeros(n, np.int32))
        used, moved = [], 0
        for s in range(n):
            before = len(self.text[s])
            p, t, i, path = self.trees[s], self.tokens[s], 0, []
            see = paths(p)
            for j in range(len(p)):      # each drafted token's attention, over the text and its own path
                way = np.nonzero(see[j])[0]
                kvs = [self.held(x, at) for at, x in enumerate(self.text[s] + [t[w] for w in way])]
                k, v = (np.array([decode(encode(y[c], "f16"), "f16") for y in kvs]) for c in (0, 1))
                o, _, off, _ = attend(q[start[s] + j][None], k, v, np.array([len(kvs) - 1]), np.ones((1, len(kvs)), bool), dim ** -0.5, 0.0, None, HALF["f16"])
                # a key's element may be one step (2^-10 of it) off where the rotation's own error turns its rounding the other way, which moves a score
                # by up to that part of the sum of its products' sizes, and a weight by as much relative to itself, the sum of the weights too
                turn = 2.0 ** -10 * dim ** -0.5 * np.einsum("hd,nhd->hn", np.abs(q[start[s] + j]), np.abs(k).repeat(h // kv, 1)).max(1)
                assert (np.abs(out[start[s] + j] - o[0]) <= off[0] + 2.02 * turn[:, None] * np.abs(v).max()).all(), (note, s, j)
            while i is not None and i < len(p):
                path.append(i)
                i = next((j for j in range(i + 1, len(p)) if p[j] == i and t[j] == self.after[t[i]]), None)
            moved += sum(a != b for a, b in enumerate(path))
            self.text[s] += [t[j] for j in path]
            assert ctx[s] == len(self.text[s]) == before + len(path), (note, s)
            blocks = table[s, :-(-len(self.text[s]) // self.BS)]
            used += blocks.tolist()
        assert len(used) == len(set(used)) and d.get(self.nfree, np.zeros(1, np.int32))[0] == self.NB - len(used), note
        for c in self.caches:
            kc, vc = (decode(d.get(x, np.zeros(self.shape, np.uint16)), "f16") for x in (c.k, c.v))
            for s in range(n):
                for at, x in enumerate(self.text[s]):
                    k, v = self.held(x, at)
                    b = table[s, at // self.BS]
                    assert (np.abs(kc[b, :, at % self.BS] - k) <= HALF["f16"] * np.abs(k) + 2.0 ** -18).all() and (vc[b, :, at % self.BS] == decode(encode(v, "f16"), "f16")).all(), (note, s, at)
        print(f"  {note}: lengths {ctx.tolist()}, {moved} rows moved", flush=True)
        return moved


def test_drafting_steps_eager_and_captured():
    """steps of a server that drafts; then one captured into a graph and replayed for other drafts, with eager steps of another server between"""
    with Dev() as d:
        s, other = Drafting(d, np.random.default_rng(1), 90), Drafting(d, np.random.default_rng(2), 70)
        moved = 0
        for i, sizes in enumerate([[20, 1, 7, 30, 3], [1, 1, 1, 1, 1], [0, 12, 5, 2, 33], [9, 9, 9, 9, 9]]):
            s.feed(sizes); s.queue()
            moved += s.check(f"step {i}")
        hip = C.CDLL("libamdhip64.so")
        stream, graph, ex = C.c_void_p(d.lib.mmoe_stream()), C.c_void_p(), C.c_void_p()
        assert hip.hipStreamBeginCapture(stream, 1) == 0
        s.queue()
        assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
        assert hip.hipGraphInstantiate(C.byref(ex), graph, None, None, C.c_size_t(0)) == 0
        try:
            for i in range(8):
                s.feed([1 + (i * 7 + j * 5) % 18 for j in range(5)])
                assert hip.hipGraphLaunch(ex, stream) == 0
                moved += s.check(f"replay {i}")
                if i % 3 == 0:
                    other.feed([3 + j for j in range(5)]); other.queue()
                    other.check(f"eager between, {i}")
        finally:
            hip.hipGraphExecDestroy(ex); hip.hipGraphDestroy(graph)
        assert moved > 5
