"""Launch shapes of the many-sequence kernels that only larger calls have: several tokens per workgroup of the rotation and more
heads than its lanes take at once, joins by 1024 threads."""
import numpy as np
import pytest

import maplemoe as M
import test_gpu_paged as base
from paged_ref import Batch, Dev, encode

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,heads,kv,dim,rot,inter,tin,tout,bs,token_major,far", [
    (2101, 16, 4, 128, 64, 0, "bf16", "bf16", 64, False, 100000),     # two tokens of 24 heads, the last workgroup has one
    (2101, 16, 4, 128, 64, 1, "f32", "f16", 16, True, 100000),
    (1031, 16, 4, 128, 128, 0, "f16", "f16", 64, False, 4096),
    (2051, 6, 2, 128, 36, 1, "f16", "f32", 32, False, 4096),           # four tokens of 10 heads, part of a unit rotated
    (4099, 4, 1, 128, 96, 0, "bf16", "bf16", 16, False, 9000),         # eight tokens of 6 heads, the last workgroup has three
    (4099, 4, 1, 64, 64, 1, "f32", "bf16", 16, False, 9000),
    (3001, 2, 1, 64, 20, 0, "f16", "f16", 16, False, 9000),            # through LDS, five tokens
    (37, 32, 32, 128, 64, 0, "f32", "f16", 16, False, 4096),           # 96 heads: two rounds of 48
    (700, 40, 8, 256, 256, 1, "bf16", "f32", 16, False, 4096),         # 56 heads of 256: three rounds of 24
    (1030, 40, 0, 128, 64, 0, "f32", "f16", 0, False, 4096),           # 40 heads, no cache
])
def test_rope_of_many_tokens_and_heads(n, heads, kv, dim, rot, inter, tin, tout, bs, token_major, far):
    base.test_rope(n, heads, kv, dim, rot, inter, tin, tout, bs, token_major, far)


@pytest.mark.parametrize("n,heads,kv,dim,rot,inter", [(1500, 6, 2, 128, 64, 0), (4101, 2, 1, 128, 128, 1), (2050, 2, 1, 64, 20, 0), (40, 64, 8, 128, 64, 0), (40, 64, 8, 128, 64, 1)])
def test_rope_in_place_of_many_tokens_and_heads(n, heads, kv, dim, rot, inter):
    print(f"\n  n={n} heads={heads}/{kv} dim={dim} rot={rot} inter={inter}", flush=True)
    rng = np.random.default_rng(n + rot)
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


@pytest.mark.parametrize("kw", [
    dict(qlens=[1], lens=[40000], dim=64, kind="f16"),                             # 157 parts
    dict(qlens=[1], lens=[70001], dim=64, kind="bf16", alibi=True),                # 274 parts
    dict(qlens=[2, 1], lens=[33100, 33025], shared=33024, dim=64, kind="f16"),     # 129 chunks of shared positions and one of each sequence's own
    dict(qlens=[1], lens=[36000], dim=128, kind="f16"),
    dict(qlens=[20], lens=[60000], dim=64, kind="bf16", heads=1),                  # 256 runs of a row tile
])
def test_a_join_of_many_parts(kw):
    kw = dict(dict(heads=2, kv=1, bs=128, width_more=0), **kw)
    b = Batch(np.random.default_rng(kw["lens"][0]), **kw)
    print(f"\n  {kw}", flush=True)
    with Dev() as d:
        a = b.upload(d)
        got = []
        for _ in range(2):
            M.check(d.lib.mmoe_attn_paged(a, b.cache), "attention")
            b.check(d, "many parts")
            got.append(d.get(b.p_out, b.out0))
        assert np.array_equal(*got)
