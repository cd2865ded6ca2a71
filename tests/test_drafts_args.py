"""Arguments that the operators for drafted tokens and shared blocks refuse (before any GPU work, so also without a GPU), and their references'
own checks."""
import numpy as np
import pytest

import maplemoe as M
from draft_ref import accept, compact, fork, free_blocks, paths, tree, tree_plan

P = 1 << 20   # stands for a device address: refused calls follow no pointer


def cache(**kw):
    return M.KvCache(**dict(dict(k=P, v=P, block_stride=4 * 16 * 128, head_stride=16 * 128, token_stride=128, nblocks=10, block_size=16, heads=4, head_dim=128,
                                 dtype=M.F16), **kw))


def attn(**kw):
    return M.PagedAttn(**dict(dict(q=P, out=P, q_token=2048, q_head=128, out_token=2048, out_head=128, qstart=P, len=P, table=P, ws=P, ws_bytes=1 << 40, nseq=2,
                                   ntok=20, heads=16, width=8, max_q=10, max_len=100, scale=0.1), **kw))


def refused(rc, word):
    assert rc == -1 and word in M.lib().mmoe_last_error(), M.lib().mmoe_last_error()


@pytest.mark.parametrize("kw,word", [
    (dict(nseq=-1), b"sequences"), (dict(nseq=4097), b"sequences"), (dict(ntok=-1), b"tokens"), (dict(ntok=(1 << 23) + 1), b"tokens"), (dict(words=0), b"words"),
    (dict(words=9), b"words"), (dict(qstart=None), b"pointer"), (dict(len=None), b"pointer"), (dict(parent=None), b"pointer"), (dict(pos=None), b"pointer"),
    (dict(bits=None), b"pointer"), (dict(bits=P + 4), b"aligned")])
def test_tree_plan_refusals(kw, word):
    refused(M.lib().mmoe_tree_plan(M.TreePlan(**dict(dict(qstart=P, len=P, parent=P, pos=P, bits=P, nseq=2, ntok=9, words=1), **kw))), word)


@pytest.mark.parametrize("kw,ckw,bits,words,word", [
    (dict(hi=P), {}, P, 1, b"hi"), ({}, {}, P, 0, b"words"), ({}, {}, P, 9, b"words"), (dict(max_q=65), {}, P, 1, b"max_q"), (dict(max_q=513), {}, P, 8, b"max_q"),
    ({}, {}, None, 1, b"pointer"), ({}, {}, P + 4, 1, b"aligned"), ({}, dict(head_dim=96), P, 1, b"head_dim"), ({}, dict(dtype=M.F32), P, 1, b"type"),
    (dict(heads=18), {}, P, 1, b"heads"), (dict(shared=8), {}, P, 1, b"shared"), (dict(window=-1), {}, P, 1, b"window"), (dict(cap=2000.0), {}, P, 1, b"cap"),
    (dict(scale=float("nan")), {}, P, 1, b"scale"), (dict(nseq=4096, ntok=1 << 18, max_q=512, width=1 << 22, max_len=1 << 26, heads=16), dict(heads=1), P, 8, b"too many"), (dict(q=None), {}, P, 1, b"pointer"), (dict(q=P + 8), {}, P, 1, b"aligned"), (dict(ws_bytes=10), {}, P, 1, b"workspace"),
    (dict(ws=P + 16), {}, P, 1, b"workspace"), (dict(max_len=129), {}, P, 1, b"max_len"), (dict(q_head=4), {}, P, 1, b"strides")])
def test_attn_tree_refusals(kw, ckw, bits, words, word):
    refused(M.lib().mmoe_attn_tree(attn(**kw), cache(**ckw), bits, words), word)
    assert b"mmoe_attn_tree" in M.lib().mmoe_last_error()


def test_attn_tree_workspace():
    lib = M.lib()
    assert lib.mmoe_attn_tree_ws(attn(), cache(), P, 1) > 0
    # it follows the tokens and the sequences, not the bound of their lengths
    assert lib.mmoe_attn_tree_ws(attn(max_len=128), cache(), P, 1) == lib.mmoe_attn_tree_ws(attn(max_len=0), cache(), P, 1)
    assert lib.mmoe_attn_tree_ws(attn(hi=P), cache(), P, 1) == 0 and lib.mmoe_attn_tree_ws(attn(), cache(), P, 0) == 0
    assert lib.mmoe_attn_tree(None, cache(), P, 1) == -1 and lib.mmoe_attn_tree(attn(), None, P, 1) == -1
    assert lib.mmoe_attn_tree(attn(ntok=0), cache(), P, 1) == 0 and lib.mmoe_attn_tree(attn(nseq=0), cache(), P, 1) == 0


@pytest.mark.parametrize("kw,word", [
    (dict(nseq=-1), b"sequences"), (dict(nseq=4097), b"sequences"), (dict(ntok=-1), b"tokens"), (dict(qstart=None), b"pointer"), (dict(len=None), b"pointer"),
    (dict(parent=None), b"pointer"), (dict(token=None), b"pointer"), (dict(next=None), b"pointer"), (dict(kept=None), b"pointer"), (dict(count=None), b"pointer"),
    (dict(ctx=None), b"pointer"), (dict(last=None), b"pointer")])
def test_accept_refusals(kw, word):
    a = dict(qstart=P, len=P, parent=P, token=P, next=P, kept=P, count=P, ctx=P, last=P, nseq=2, ntok=9)
    refused(M.lib().mmoe_tree_accept(M.TreeAccept(**dict(a, **kw))), word)


def layers(n, other=None, **kw):
    c = (M.KvCache * n)(*(cache(**kw) for _ in range(n)))
    if other:
        c[n - 1] = cache(**dict(kw, **other))
    return c


@pytest.mark.parametrize("other", [dict(block_stride=8 * 16 * 128), dict(head_stride=0), dict(token_stride=256), dict(nblocks=9), dict(block_size=32), dict(heads=2), dict(head_dim=64),
                                   dict(dtype=M.BF16)])
def test_layers_must_be_alike(other):
    refused(M.lib().mmoe_kv_compact(M.KvCompact(table=P, first=P, count=P, kept=P, nseq=1, width=4, nkept=5), layers(3, other), 3), b"layer 2")
    refused(M.lib().mmoe_kv_copy(M.KvCopy(copy_from=P, copy_to=P, ncopy=1), layers(3, other), 3), b"layer 2")


@pytest.mark.parametrize("kw,n,ckw,word", [
    (dict(nseq=-1), 1, {}, b"sequences"), (dict(nseq=4097), 1, {}, b"sequences"), (dict(width=0), 1, {}, b"tables"), (dict(nkept=-1), 1, {}, b"kept"), (dict(nkept=(1 << 30) + 1), 1, {}, b"kept"),
    (dict(table=None), 1, {}, b"pointer"), (dict(first=None), 1, {}, b"pointer"), (dict(count=None), 1, {}, b"pointer"), (dict(kept=None), 1, {}, b"pointer"),
    ({}, 0, {}, b"layers"), ({}, 129, {}, b"layers"), ({}, 1, dict(head_dim=12), b"head_dim"), ({}, 1, dict(head_dim=264, token_stride=264), b"head_dim"), ({}, 1, dict(k=None), b"set"),
    ({}, 1, dict(block_size=20), b"block size"), ({}, 1, dict(v=P + 8), b"aligned"), (dict(nseq=4096), 128, dict(heads=1024), b"too many")])
def test_compact_refusals(kw, n, ckw, word):
    a = M.KvCompact(**dict(dict(table=P, first=P, count=P, kept=P, nseq=2, width=4, nkept=9), **kw))
    refused(M.lib().mmoe_kv_compact(a, layers(max(n, 1), **ckw), n), word)


@pytest.mark.parametrize("kw,n,ckw,word", [
    (dict(ncopy=-1), 1, {}, b"copies"), (dict(ncopy=4097), 1, {}, b"copies"), (dict(copy_from=None), 1, {}, b"pointer"), (dict(copy_to=None), 1, {}, b"pointer"), ({}, 0, {}, b"layers"),
    ({}, 129, {}, b"layers"), ({}, 1, dict(head_dim=4), b"head_dim"), (dict(ncopy=4096), 128, dict(heads=1024, block_size=1024), b"too many")])
def test_copy_refusals(kw, n, ckw, word):
    a = M.KvCopy(**dict(dict(copy_from=P, copy_to=P, ncopy=2), **kw))
    refused(M.lib().mmoe_kv_copy(a, layers(max(n, 1), **ckw), n), word)


TABLES = [(dict(block_size=24), b"block size"), (dict(nseq=-1), b"sequences"), (dict(nseq=4097), b"sequences"), (dict(nblocks=-1), b"blocks"), (dict(nblocks=1 << 28), b"blocks"),
          (dict(width=0), b"tables"), (dict(width=1 << 27), b"tables"), (dict(shared=8), b"shared"), (dict(shared=-16), b"shared"), (dict(shared=80), b"shared"),
          (dict(nfree=None), b"pointer"), (dict(nfree_out=None), b"pointer"), (dict(ctx=None), b"pointer"), (dict(table=None), b"pointer"), (dict(free_list=None), b"pointer")]


@pytest.mark.parametrize("kw,word", TABLES + [(dict(nfork=-1), b"forks"), (dict(nfork=4097), b"forks")] + [
    (dict([(k, None)]), b"pointer") for k in ("src", "dst", "ctx_out", "table_out", "holders", "copy_from", "copy_to", "copy_count")])
def test_fork_refusals(kw, word):
    a = dict(src=P, dst=P, ctx=P, table=P, ctx_out=P, table_out=P, holders=P, free_list=P, nfree=P, nfree_out=P, copy_from=P, copy_to=P, copy_count=P, nfork=2, nseq=2,
             width=4, nblocks=10, block_size=16)
    refused(M.lib().mmoe_kv_fork(M.KvFork(**dict(a, **kw))), word)


@pytest.mark.parametrize("kw,word", TABLES + [(dict(keep=None), b"pointer"), (dict(len=None), b"pointer"), (dict(nseq=4096, width=(1 << 18) + 1), b"places")])
def test_free_refusals(kw, word):
    a = dict(ctx=P, keep=P, table=P, nfree=P, len=P, free_list=P, nfree_out=P, nseq=2, width=4, nblocks=10, block_size=16)
    refused(M.lib().mmoe_kv_free(M.KvFree(**dict(a, **kw))), word)


def test_missing_arguments():
    lib = M.lib()
    for f in (lib.mmoe_tree_plan, lib.mmoe_tree_accept, lib.mmoe_kv_fork, lib.mmoe_kv_free):
        refused(f(None), b"no arguments")
    refused(lib.mmoe_kv_compact(None, layers(1), 1), b"no arguments")
    refused(lib.mmoe_kv_compact(M.KvCompact(), None, 1), b"no arguments")
    refused(lib.mmoe_kv_copy(None, layers(1), 1), b"no arguments")
    refused(lib.mmoe_kv_copy(M.KvCopy(), None, 1), b"no arguments")


# ---------------------------------------------------------------------------------------------------- the references, on cases worked out by hand
def test_reference_tree_and_walk():
    #      0
    #    1   2
    #   3 4   5
    #   6
    parent = [-1, 0, 0, 1, 1, 2, 3]
    a = paths(parent)
    assert np.nonzero(a[6])[0].tolist() == [0, 1, 3, 6] and np.nonzero(a[5])[0].tolist() == [0, 2, 5]
    pos, bits = tree_plan([0, 7], [107], parent, 1, 8)
    assert pos.tolist() == [100, 101, 101, 102, 102, 102, 103, 0] and bits[6, 0] == 0b1001011 and bits[7, 0] == 0
    token, choice = [9, 5, 5, 7, 8, 8, 1], [5, 8, 0, 0, 44, 0, 0]   # 5 behind 0: node 1 (the lower); 8 behind it: node 4
    kept, count, ctx, last = accept([0, 7], [107], parent, token, choice, np.full(7, -1))
    assert kept.tolist() == [100, 101, 104, -1, -1, -1, -1] and (count[0], ctx[0], last[0]) == (3, 103, 44)
    assert tree(np.random.default_rng(0), 5, 1) == [-1, 0, 1, 2, 3]


def test_reference_compact_fork_free():
    cache_ = np.arange(4 * 16).reshape(4, 16, 1)
    got = compact(cache_, np.array([[2, 0]]), [0], [4], np.array([14, 16, 18, 31]), 4, 16)
    assert got[2, 14:, 0].tolist() == [46, 0] and got[0, :3, 0].tolist() == [2, 15, 2]
    table = np.array([[5, 6, 7, -1], [-1] * 4, [-1] * 4])
    f = fork([0, 0], [1, 2], [40, 16], np.array([40, 0, 0]), np.array([40, 0, 0]), table, table, np.zeros(9, int), np.arange(9), 2, 16, 0, 9)
    assert f["table_out"].tolist() == [[5, 6, 7, -1], [5, 6, 1, -1], [5, -1, -1, -1]] and f["holders"].tolist() == [0, 0, 0, 0, 0, 2, 1, 0, 0]
    assert (f["copy_from"].tolist(), f["copy_to"].tolist(), f["copy_count"].tolist(), f["nfree_out"][0]) == ([7, -1], [1, -1], [8, 0], 1)
    r = free_blocks(np.array([40, 40, 16]), [0, 20, 0], f["table_out"], f["holders"], np.full(9, -1), 0, 16, 0, 9)
    # row 0 ends: 7 goes back, 5 and 6 lose a holder; row 1 would end inside 6, which row 0 holds as the call begins: it stays whole; row 2 drops 5
    assert r["len"].tolist() == [0, 40, 0] and r["holders"].tolist() == [0] * 9 and r["free_list"][:1].tolist() == [7] and r["nfree_out"][0] == 1
