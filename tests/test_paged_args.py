"""Arguments that the many-sequence operators refuse (before any GPU work, so also without a GPU), and the rotation frequencies."""
import numpy as np
import pytest

import maplemoe as M

P = 1 << 20   # stands for a device address: refused calls follow no pointer


def cache(**kw):
    return M.KvCache(**dict(dict(k=P, v=P, block_stride=4 * 16 * 128, head_stride=16 * 128, token_stride=128, nblocks=10, block_size=16, heads=4, head_dim=128,
                                 dtype=M.F16), **kw))


def attn(**kw):
    return M.PagedAttn(**dict(dict(q=P, out=P, q_token=2048, q_head=128, out_token=2048, out_head=128, qstart=P, len=P, table=P, ws=P, ws_bytes=1 << 40, nseq=2,
                                   ntok=2, heads=16, width=8, max_q=1, max_len=100, scale=0.1), **kw))


def rope(**kw):
    return M.Rope(**dict(dict(q=P, k=P, v=P, q_out=P, q_token=2048, q_head=128, k_token=2048, k_head=128, v_token=2048, v_head=128, qo_token=2048, qo_head=128,
                              pos=P, slot=P, freq=P, ntok=2, heads=16, kv_heads=4, head_dim=128, rot=64, in_dtype=M.F32, out_dtype=M.F16, mag=1.0), **kw))


def plan(**kw):
    return M.KvPlan(**dict(dict(ctx=P, add=P, table=P, free_list=P, nfree=P, nfree_out=P, len=P, qstart=P, pos=P, slot=P, nseq=2, width=4, nblocks=10, block_size=16,
                                ntok=2), **kw))


def refused(rc, word):
    assert rc == -1 and word in M.lib().mmoe_last_error(), M.lib().mmoe_last_error()


@pytest.mark.parametrize("kw,word", [
    (dict(block_size=0), b"block size"), (dict(block_size=24), b"block size"), (dict(block_size=8), b"block size"), (dict(block_size=2048), b"block size"),
    (dict(nseq=-1), b"sequences"), (dict(nseq=4097), b"sequences"), (dict(ntok=-1), b"tokens"), (dict(nblocks=-1), b"blocks"), (dict(nblocks=1 << 28), b"blocks"),
    (dict(width=0), b"tables"), (dict(width=1 << 28), b"tables"), (dict(width=(1 << 26) + 1), b"tables"), (dict(ntok=(1 << 23) + 1), b"tokens"), (dict(shared=8), b"shared"), (dict(shared=-16), b"shared"), (dict(shared=80), b"shared"),
    (dict(ctx=None), b"pointer"), (dict(add=None), b"pointer"), (dict(table=None), b"pointer"), (dict(free_list=None), b"pointer"), (dict(nfree=None), b"pointer"),
    (dict(nfree_out=None), b"pointer"), (dict(len=None), b"pointer"), (dict(qstart=None), b"pointer"), (dict(pos=None), b"pointer"), (dict(slot=None), b"pointer")])
def test_plan_refusals(kw, word):
    refused(M.lib().mmoe_kv_plan(plan(**kw)), word)


@pytest.mark.parametrize("kw,ckw,word", [
    (dict(in_dtype=3), {}, b"types"), (dict(out_dtype=-1), {}, b"types"), (dict(head_dim=12), {}, b"head_dim"), (dict(head_dim=264), {}, b"head_dim"),
    (dict(rot=63), {}, b"rotated"), (dict(rot=130), {}, b"rotated"), (dict(rot=-2), {}, b"rotated"), (dict(ntok=-1), {}, b"tokens"), (dict(ntok=(1 << 23) + 1), {}, b"tokens"), (dict(heads=-1), {}, b"heads"),
    (dict(mag=float("nan")), {}, b"mag"), (dict(out_dtype=M.BF16), {}, b"cache of"), (dict(kv_heads=2), {}, b"cache of"), (dict(head_dim=64), {}, b"cache of"),
    ({}, dict(block_size=20), b"block size"), ({}, dict(k=P + 8), b"aligned"), ({}, dict(v=None), b"set"), ({}, dict(nblocks=0), b"blocks"), ({}, dict(nblocks=1 << 27), b"blocks"),
    ({}, dict(dtype=7), b"type"), ({}, dict(heads=0), b"heads"), ({}, dict(token_stride=132), b"strides"), ({}, dict(head_stride=-8), b"strides"),
    (dict(pos=None), {}, b"pointer"), (dict(freq=None), {}, b"pointer"), (dict(q=None), {}, b"pointer"), (dict(q_out=None), {}, b"pointer"), (dict(k=None), {}, b"pointer"),
    (dict(v=None), {}, b"pointer"), (dict(slot=None), {}, b"pointer"), (dict(q=P + 4), {}, b"aligned"), (dict(q_out=P + 2), {}, b"aligned"), (dict(v_token=2047), {}, b"strides")])
def test_rope_refusals(kw, ckw, word):
    refused(M.lib().mmoe_rope_kv(rope(**kw), cache(**ckw)), word)


def test_rope_without_a_cache_wants_k_out():
    refused(M.lib().mmoe_rope_kv(rope(), None), b"pointer")
    refused(M.lib().mmoe_rope_kv(None, None), b"no arguments")
    refused(M.lib().mmoe_kv_plan(None), b"no arguments")


ATTN = [
    (dict(heads=6), {}, b"query heads"), (dict(heads=0), {}, b"query heads"), (dict(nseq=-1), {}, b"sequences"), (dict(nseq=5000), {}, b"sequences"), (dict(ntok=-1), {}, b"tokens"),
    (dict(ntok=1 << 28), {}, b"tokens"), (dict(width=0), {}, b"tables"), (dict(width=1 << 27), {}, b"tables"), (dict(max_q=-1), {}, b"max_q"), (dict(max_len=-1), {}, b"max_len"),
    (dict(max_len=129), {}, b"max_len"), (dict(shared=8), {}, b"shared"), (dict(shared=-16), {}, b"shared"), (dict(shared=112), {}, b"shared"), (dict(window=-1), {}, b"window"),
    (dict(scale=float("inf")), {}, b"scale"), (dict(scale=0.0), {}, b"scale"), (dict(scale=-0.1), {}, b"scale"), (dict(cap=-1.0), {}, b"cap"), (dict(cap=float("nan")), {}, b"cap"), (dict(cap=1025.0), {}, b"cap"),
    (dict(cap=1e-39), {}, b"cap"), (dict(ntok=(1 << 22) + 1, heads=256), {}, b"tokens"), (dict(q_head=4), {}, b"strides"), (dict(out_token=-8), {}, b"strides"),
    ({}, dict(dtype=M.F32), b"cache type"), ({}, dict(token_stride=(1 << 26) + 8), b"stride"), ({}, dict(head_dim=96), b"head_dim"), ({}, dict(head_dim=256, token_stride=256), b"head_dim"), ({}, dict(token_stride=120), b"stride"), ({}, dict(block_size=17), b"block size"),
    ({}, dict(k=None), b"set"), ({}, dict(nblocks=0), b"blocks")]


@pytest.mark.parametrize("kw,ckw,word", ATTN)
def test_attention_refusals(kw, ckw, word):
    lib = M.lib()
    refused(lib.mmoe_attn_paged(attn(**kw), cache(**ckw)), word)
    assert lib.mmoe_attn_paged_ws(attn(**kw), cache(**ckw)) == 0


@pytest.mark.parametrize("kw,word", [(dict(q=None), b"pointer"), (dict(out=None), b"pointer"), (dict(qstart=None), b"pointer"), (dict(len=None), b"pointer"),
                                     (dict(table=None), b"pointer"), (dict(q=P + 8), b"aligned"), (dict(out=P + 2), b"aligned"), (dict(ws=None), b"workspace"),
                                     (dict(ws=P + 16), b"workspace"), (dict(ws_bytes=0), b"workspace"),
                                     (dict(nseq=4096, width=1 << 26, max_len=1 << 30, heads=2048), b"key/value heads"), (dict(nseq=4096, width=1 << 26, max_len=1 << 30), b"too many")])
def test_attention_refusals_of_pointers(kw, word):
    refused(M.lib().mmoe_attn_paged(attn(**kw), cache(heads=2048) if word == b"key/value heads" else cache(heads=16) if word == b"too many" else cache()), word)


def test_nothing_to_do_is_no_error():
    lib = M.lib()
    assert lib.mmoe_attn_paged(attn(nseq=0), cache()) == 0 and lib.mmoe_attn_paged(attn(ntok=0), cache()) == 0
    assert lib.mmoe_rope_kv(rope(ntok=0), cache()) == 0 and lib.mmoe_rope_kv(rope(heads=0, kv_heads=0), None) == 0
    refused(lib.mmoe_attn_paged(None, None), b"no arguments")


def freqs(*a):
    f = np.zeros(a[0] // 2)
    assert M.lib().mmoe_rope_freqs(*a, M.ptr(f)) == 0
    return f


def test_rope_frequencies():
    i = np.arange(32)
    plain = 10000.0 ** (-2.0 * i / 64)
    assert np.allclose(freqs(64, 10000.0, 1.0, 0, 0.0, 0.0), plain, rtol=1e-15, atol=0)
    assert np.allclose(freqs(64, 10000.0, 8.0, 0, 0.0, 0.0), plain / 8, rtol=1e-15, atol=0)
    f = freqs(64, 10000.0, 8.0, 4096, 1.0, 32.0)
    turns = 4096 * plain / (2 * np.pi)
    assert np.allclose(f[turns >= 32], plain[turns >= 32], rtol=1e-15, atol=0) and np.allclose(f[turns <= 1], plain[turns <= 1] / 8, rtol=1e-15, atol=0)
    mid = (turns > 1) & (turns < 32)
    g = (turns[mid] - 1) / 31
    assert mid.any() and np.allclose(f[mid], plain[mid] * (g + (1 - g) / 8), rtol=1e-14, atol=0)
    assert (np.diff(f) < 0).all()


@pytest.mark.parametrize("a", [(63, 1e4, 1.0, 0, 1.0, 32.0), (-2, 1e4, 1.0, 0, 1.0, 32.0), (258, 1e4, 1.0, 0, 1.0, 32.0), (64, 1.0, 1.0, 0, 1.0, 32.0), (64, float("nan"), 1.0, 0, 1.0, 32.0),
                               (64, 1e4, 0.5, 0, 1.0, 32.0), (64, 1e4, float("inf"), 0, 1.0, 32.0), (64, 1e4, 2.0, -1, 1.0, 32.0), (64, 1e4, 2.0, 10, 32.0, 32.0), (64, 1e4, 2.0, 10, -1.0, 32.0)])
def test_rope_frequencies_refused(a):
    f = np.zeros(200)
    refused(M.lib().mmoe_rope_freqs(*a, M.ptr(f)), b"mmoe_rope_freqs")
    refused(M.lib().mmoe_rope_freqs(64, 1e4, 1.0, 0, 1.0, 32.0, None), b"output")
