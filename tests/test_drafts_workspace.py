"""What mmoe_attn_tree's workspace depends on (no GPU needed)."""
import pytest

import maplemoe as M
from test_drafts_args import P, attn, cache, refused


def size(ckw={}, words=1, **kw):
    return M.lib().mmoe_attn_tree_ws(attn(**kw), cache(**ckw), P, words)


@pytest.mark.parametrize("kw,ckw", [(dict(nseq=64, ntok=256, max_q=4), {}), (dict(nseq=48, ntok=192, max_q=4), {}), (dict(nseq=200, ntok=800, max_q=4), {}), (dict(nseq=32, ntok=2048, max_q=64), {}),
                                    (dict(nseq=64, ntok=200, max_q=5, heads=8), dict(head_dim=64, heads=8)), (dict(nseq=2), {})])
def test_one_workspace_serves_every_bound_and_window(kw, ckw):
    """few positions and many row tiles stay whole and need no results, the same call with a larger bound does: both have the same room"""
    kw = dict(kw, width=1024)
    want = size(ckw, **kw, max_len=16384)
    for max_len in (0, 1, 63, 64, 700, 703, 704, 767, 768, 769, 4096, 16384):
        for window in (0, 1, 100, 512, 4096):
            assert size(ckw, **kw, max_len=max_len, window=window) == want, (max_len, window)
    # and a call for which it is too small is refused whatever its bounds
    for max_len in (64, 700, 4096):
        refused(M.lib().mmoe_attn_tree(attn(**kw, max_len=max_len, ws_bytes=want - 1), cache(**ckw), P, 1), b"workspace")


@pytest.mark.parametrize("ckw,heads", [({}, 16), (dict(heads=1), 4), (dict(heads=8, head_dim=64), 8), (dict(heads=1, head_dim=64), 64)])
@pytest.mark.parametrize("shared", [0, 64])
def test_it_grows_with_tokens_and_sequences(ckw, heads, shared):
    """a workspace for more tokens, larger trees or more sequences serves fewer; one with shared positions serves layers without them"""
    def at(nseq, ntok, max_q, sh=shared):
        return size(ckw, nseq=nseq, ntok=ntok, max_q=max_q, heads=heads, width=64, max_len=1000, shared=sh)
    seqs, toks, most = (1, 2, 63, 64, 65, 70, 300, 4096), (1, 60, 400, 5000, 100000), (1, 2, 9, 33, 64)
    for n in seqs:
        for t in toks:
            for q in most:
                x = at(n, t, q)
                assert x and x == at(n, t, q) and at(n, t, q, 0) <= x == at(n, t, q, 4 * shared)
                assert all(at(m, t, q) <= x for m in seqs if m < n) and all(at(n, u, q) <= x for u in toks if u < t) and all(at(n, t, r) <= x for r in most if r < q), (n, t, q)


@pytest.mark.parametrize("kw,ckw", [(dict(nseq=4096, ntok=1 << 18, max_q=512, width=1 << 22, max_len=1 << 26, heads=16), dict(heads=1)),
                                    (dict(nseq=64, ntok=1 << 20, max_q=512, width=1 << 26, max_len=1 << 30, heads=1024), dict(heads=1))])
def test_no_size_for_what_is_too_much_for_a_launch(kw, ckw):
    refused(M.lib().mmoe_attn_tree(attn(**kw), cache(**ckw), P, 8), b"too many")
    M.lib().mmoe_attn_tree(None, cache(), P, 1)      # another message
    assert M.lib().mmoe_attn_tree_ws(attn(**kw), cache(**ckw), P, 8) == 0 and b"too many" in M.lib().mmoe_last_error()
    assert M.lib().mmoe_attn_tree_ws(attn(**dict(kw, max_len=1000)), cache(**ckw), P, 8) > 0


@pytest.mark.parametrize("shared", [0, 2048])
def test_sequences_at_rest_take_no_room(shared):
    """64 drafts of 20 tokens in a batch of 4096: what is kept follows the tokens. Of each of 4 key/value heads 5120 rows over the shared positions and of
    their own (1280 sequences of one token at the worst), and 128 pieces of 128 rows that a cut adds, 520 bytes a row and head"""
    at = size(nseq=4096, ntok=1280, max_q=20, width=512, max_len=8192, shared=shared)
    waves = 128 * 4 + 160 + 160 + 1280 if shared else 128 * 3 + 160 + 1280
    assert at <= waves * 32 * 4 * 520 + 4096 * 64 and at < (142e6 if shared else 52e6)
    assert at <= size(nseq=1280, ntok=1280, max_q=20, width=512, max_len=8192, shared=shared)


def test_words_with_the_window_along_the_path():
    W = M.TREE_WINDOW
    assert size(window=9, words=1 | W) == size(window=9) and size(words=8 | W) > 0
    for words in (W, 9 | W, 2 * W | 1, -1, 1 - W):
        refused(M.lib().mmoe_attn_tree(attn(), cache(), P, words), b"words")
    refused(M.lib().mmoe_attn_tree(attn(max_q=65), cache(), P, 1 | W), b"max_q")
