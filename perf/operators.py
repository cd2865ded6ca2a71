"""Performance cases of the operators that serve many sequences at once: block tables, rotary positions, paged attention.

Kinds of case (a case is a dict of plain values; `kind` says which operator it calls):

  plan    block tables and slot maps of one step, from the requests' lengths (mmoe_kv_plan): finished sequences give their
          blocks back, the others get blocks for their new tokens; positions and slots of every token.
  rope    rotary positions of a step's queries and keys, and the write of its keys and values into the blocks (mmoe_rope_kv).
  attn    attention of a step's queries over the blocks (mmoe_attn_paged): a batch that shares a prefix (`shared` > 0, held
          in blocks that every table begins with), scores capped by a tanh (`cap`), a bias that falls with the distance
          (`alibi`), a sliding window, documents packed into one sequence (`docs`: each token sees its own document only),
          a prefix that every query sees whole (`prefix`).

The lengths of a case's sequences are a fixed ragged pattern between two bounds; a seed shuffles them and changes every value.
Caches are [block][key/value head][position in the block][dim]. The heads are Maple's (16 query and 4 key/value heads of 128,
64 rotated dims, window 512) or generic.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------------------------------- cases
def _plan(nseq, add, ctx, bs, shared=0, done=0, tight=False, pad=0):
    return dict(kind="plan", nseq=nseq, add=add, ctx=ctx, bs=bs, shared=shared, done=done, tight=tight, pad=pad)


def _rope(n, tin, tout, heads=16, kv=4, dim=128, rot=64, inter=False, scaled=False, bs=16, step=False, far=4096):
    return dict(kind="rope", n=n, tin=tin, tout=tout, heads=heads, kv=kv, dim=dim, rot=rot, inter=inter, scaled=scaled, bs=bs, step=step, far=far)


def _attn(nseq, q, ctx, shared=0, type="bf16", heads=16, kv=4, dim=128, bs=16, cap=0.0, alibi=False, window=0, docs=0, prefix=0.0):
    return dict(kind="attn", nseq=nseq, q_lo=q[0], q_hi=q[1], ctx_lo=ctx[0], ctx_hi=ctx[1], shared=shared, type=type, heads=heads, kv=kv, dim=dim,
                bs=bs, cap=cap, alibi=alibi, window=window, docs=docs, prefix=prefix)


def listed():
    return [
        # a decode step's tables: 64 sequences, one token each, three of them finished
        dict(_plan(64, 1, 3000, 16, done=3), name="plan_step_64"),
        # prompts of many lengths admitted at once, after a common prefix, into a padded batch
        dict(_plan(301, 400, 0, 64, shared=1024, pad=77), name="plan_prompts_301"),
        # a decode step of 64 sequences: Maple's heads, keys and values rounded to fp16
        dict(_rope(64, "f32", "f16", step=True), name="rope_step_64"),
        # an odd chunk of a prompt in the interleaved layout, the whole head rotated, frequencies scaled for a long context
        dict(_rope(777, "f16", "f16", rot=128, inter=True, scaled=True, bs=32, far=120000), name="rope_chunk_777"),
        # a long prompt in bf16, half layout on part of the head
        dict(_rope(8191, "bf16", "bf16", bs=64), name="rope_prompt_8191"),
        # a few sequences over a common system prompt: the latency end
        dict(_attn(7, (1, 1), (3, 90), shared=2048, type="f16"), name="shared_7"),
        # a decode batch over a long common document
        dict(_attn(64, (1, 1), (1, 500), shared=16384), name="shared_64"),
        # many sequences over a very long one, a few new tokens each (drafted tokens to verify)
        dict(_attn(96, (1, 4), (20, 700), shared=40000, bs=32), name="shared_96_long"),
        # one token of a single long sequence, with a distance bias
        dict(_attn(1, (1, 1), (99999, 99999), type="f16", alibi=True), name="alibi_step_1"),
        # prompts whose first part is seen whole by every query, each query head with its own keys, heads of 64
        dict(_attn(5, (300, 1100), (0, 0), type="f16", heads=12, kv=12, dim=64, prefix=0.3), name="prefix_prompts_5"),
        # documents packed into one long prompt, within Maple's window
        dict(_attn(1, (8191, 8191), (0, 0), window=512, docs=1500, bs=64), name="docs_8191"),
        # a chunk of a long prompt with capped scores
        dict(_attn(1, (4096, 4096), (12000, 12000), cap=30.0, bs=64), name="cap_chunk_4096"),
    ]


def _log(rng, lo, hi):
    return min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["plan", "rope", "rope", "shared", "shared", "shared", "scores", "scores", "scores", "scores"])
    bs = rng.choice([16, 16, 32, 64])
    if kind == "plan":
        nseq = _log(rng, 1, 400)
        add = rng.choice([1, 1, _log(rng, 2, 500)])
        shared = bs * rng.choice([0, 0, _log(rng, 1, 40)])
        return _plan(nseq, add, _log(rng, 1, 8000), bs, shared=shared, done=rng.randint(0, max(1, nseq // 8)) if nseq > 1 else 0,
                     tight=rng.random() < 0.25, pad=rng.choice([0, _log(rng, 1, 200)]))
    if kind == "rope":
        dim = rng.choice([64, 128, 128])
        kv = rng.choice([1, 2, 4, 8])
        tin, tout = rng.choice([("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
        return _rope(_log(rng, 1, 8191), tin, tout, heads=kv * rng.choice([1, 3, 4, 6]), kv=kv, dim=dim, rot=rng.choice([dim, dim // 2, 20]),
                     inter=rng.random() < 0.5, scaled=rng.random() < 0.4, bs=bs, step=rng.random() < 0.4, far=_log(rng, 4096, 1000000))
    kv = rng.choice([1, 2, 4, 4, 8])
    heads, dim, type = kv * rng.choice([1, 2, 3, 4, 4, 4, 8]), rng.choice([64, 128, 128]), rng.choice(["f16", "bf16"])
    while heads > 32:
        heads -= kv
    more = dict(type=type, heads=heads, kv=kv, dim=dim, bs=bs)
    if kind == "shared":
        nseq = _log(rng, 2, 96)
        return _attn(nseq, (1, rng.choice([1, 1, 1, 5])), (1, _log(rng, 4, 700)), shared=bs * (_log(rng, 256, 20000) // bs), **more,
                     cap=rng.choice([0.0, 0.0, 25.0]), alibi=rng.random() < 0.2)
    more.update(cap=rng.choice([0.0, 0.0, 20.0, 50.0]), alibi=rng.random() < 0.35, window=rng.choice([0, 0, _log(rng, 32, 2000)]))
    if rng.random() < 0.4:   # single tokens
        nseq = _log(rng, 1, 64)
        hi = _log(rng, 16, max(17, 100000 // nseq))
        return _attn(nseq, (1, 1), (rng.randint(0, hi), hi), **more)
    nseq = _log(rng, 1, 12)
    hi = _log(rng, 2, 4096 // nseq)
    ctx = rng.choice([0, 0, _log(rng, 1, 3000)])
    shape = rng.choice(["", "", "docs", "prefix"])
    return _attn(nseq, (rng.randint(1, hi), hi), (ctx // 2, ctx), **more, docs=_log(rng, 30, 1500) if shape == "docs" else 0,
                 prefix=round(rng.uniform(0.1, 0.7), 2) if shape == "prefix" else 0.0)


def _ragged(n, lo, hi):
    """n lengths between lo and hi, spread evenly and out of order"""
    return [lo + int((hi - lo + 1) * ((i + 0.5) * 0.6180339887498949 % 1.0)) for i in range(n)]


def _up(a, b):
    return -(-a // b)


# ---------------------------------------------------------------------------------------------------- inputs
def _gen(seed, *key):
    g = torch.Generator(device="cuda")
    s = int(seed)
    for k in key:
        s = (s * 1000003 + int(k) + 12345) % (1 << 62)
    g.manual_seed(s)
    return g


def _normal(g, shape, type):
    return torch.randn(shape, device="cuda", generator=g, dtype=torch.float32).to(TYPES[type])


def _ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()


def _lens(case):
    """(cached, new) lengths of a plan case's sequences; the finished ones bring no new tokens"""
    n = case["nseq"]
    ctx = [case["shared"] + c for c in _ragged(n, 0, case["ctx"])]
    add = _ragged(n, 1, case["add"])
    return ctx, [0 if i < case["done"] else a for i, a in enumerate(add)]


def _prepare_plan(case, seed):
    r = np.random.RandomState(seed % (1 << 32))
    n, bs, shared = case["nseq"], case["bs"], case["shared"]
    ctx, add = (np.array(v) for v in _lens(case))
    done = (np.arange(n) < case["done"]).astype(np.int32)
    order = r.permutation(n)
    ctx, add, done = ctx[order], add[order], done[order]
    keep, held = shared // bs, -(-ctx // bs)
    need = int((-(-(ctx + add) // bs) - held).sum())
    used = keep + int((held - keep).sum())
    nfree = max(0, int(need * 0.7) - int(((held - keep) * done).sum())) if case["tight"] else need + 50
    nblocks = used + nfree
    width = int((-(-(ctx + add) // bs)).max()) + 3
    ids = r.permutation(nblocks)
    table = np.full((n, width), -1, np.int32)
    table[:, :keep] = ids[:keep]
    at = keep
    for s in range(n):
        table[s, keep:held[s]] = ids[at:at + held[s] - keep]
        at += held[s] - keep
    free = np.full(nblocks, -1, np.int32)
    free[:nfree] = ids[at:]
    ntok = int(add.sum()) + case["pad"]
    z = lambda *shape: torch.zeros(shape, dtype=torch.int32, device="cuda")  # noqa: E731
    return dict(kind="plan", n=n, bs=bs, shared=shared, width=width, nblocks=nblocks, ntok=ntok, ctx=_ints(ctx), add=_ints(add), done=_ints(done),
                table=_ints(table), free=_ints(free), nfree=_ints([nfree]), nfree_out=z(1), len=z(n), qstart=z(n + 1), pos=z(ntok), slot=z(ntok))


def _freqs(rot, scaled):
    """radians per position, in 64 bits; scaled: a context 8 times the 8192 positions trained on, by parts"""
    i = torch.arange(rot // 2, dtype=torch.float64)
    f = 10000.0 ** (-2.0 * i / rot)
    if scaled:
        turns = 8192 * f / (2 * math.pi)
        part = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        f = f * part + f / 8.0 * (1 - part)
    return f


def _prepare_rope(case, seed):
    g, r = _gen(seed, 1), np.random.RandomState(seed % (1 << 32))
    n, bs, dim, kv, heads = case["n"], case["bs"], case["dim"], case["kv"], case["heads"]
    if case["step"]:     # one token of each of n sequences: far positions, blocks of their own
        pos = r.randint(0, case["far"], n)
        slot = r.permutation(n) * bs + pos % bs
        nblocks = n
    else:                # a run of one sequence's positions
        pos = r.randint(0, max(1, case["far"] - n)) // bs * bs + 5 + np.arange(n)
        nblocks = _up(n + 5, bs)
        slot = r.permutation(nblocks)[(5 + np.arange(n)) // bs] * bs + pos % bs
    cache = lambda k: _normal(_gen(seed, k), (nblocks, kv, bs, dim), case["tout"])  # noqa: E731
    return dict(kind="rope", n=n, bs=bs, dim=dim, kv=kv, heads=heads, rot=case["rot"], inter=case["inter"], mag=1.2 if case["scaled"] else 1.0,
                tin=case["tin"], tout=case["tout"], qkv=_normal(g, (n, heads + 2 * kv, dim), case["tin"]), pos=_ints(pos), slot=_ints(slot),
                freq=_freqs(case["rot"], case["scaled"]).cuda(), q=torch.zeros((n, heads, dim), dtype=TYPES[case["tout"]], device="cuda"),
                k_cache=cache(2), v_cache=cache(3))


def _seqs(case):
    """(new, whole) lengths of an attn case's sequences"""
    new = _ragged(case["nseq"], case["q_lo"], case["q_hi"])
    return new, [case["shared"] + c + q for c, q in zip(reversed(_ragged(case["nseq"], case["ctx_lo"], case["ctx_hi"])), new)]


def _doc_starts(docs, n):
    """first position of each position's document, for documents of about 30 .. docs positions packed one behind the other"""
    size, starts, at = _ragged(n, min(30, docs), docs), [], 0
    for k in size:
        starts += [at] * k
        at += k
        if at >= n:
            break
    return starts[:n]


def _limits(case, q, n):
    """(lo, hi) of the q last positions of a sequence of n: the positions lo .. hi - 1 are the ones a mask leaves"""
    pos = np.arange(n - q, n)
    lo, hi = np.zeros(q, np.int64), pos + 1
    if case["docs"]:
        lo = np.array(_doc_starts(case["docs"], n))[n - q:]
    if case["prefix"]:
        hi = np.maximum(hi, int(case["prefix"] * n))
    return lo, hi


def _prepare_attn(case, seed):
    r = np.random.RandomState(seed % (1 << 32))
    new, whole = (np.array(v) for v in _seqs(case))
    order = r.permutation(case["nseq"])
    new, whole = new[order], whole[order]
    bs, shared, n, ntok = case["bs"], case["shared"], case["nseq"], int(new.sum())
    keep, held = shared // bs, -(-whole // bs)
    nblocks = keep + int((held - keep).sum()) + 1
    ids = r.permutation(nblocks)
    table = np.zeros((n, int(held.max())), np.int32)
    table[:, :keep] = ids[:keep]
    at = keep
    for s in range(n):
        table[s, keep:held[s]] = ids[at:at + held[s] - keep]
        at += held[s] - keep
    lim = [_limits(case, int(q), int(w)) for q, w in zip(new, whole)]
    cache = lambda k: _normal(_gen(seed, k), (nblocks, case["kv"], bs, case["dim"]), case["type"])  # noqa: E731
    heads = case["heads"]
    return dict(kind="attn", n=n, bs=bs, dim=case["dim"], kv=case["kv"], heads=heads, shared=shared, ntok=ntok, width=table.shape[1], type=case["type"],
                cap=case["cap"], window=case["window"], max_q=int(new.max()), max_len=int(whole.max()), scale=case["dim"] ** -0.5,
                q=(_normal(_gen(seed, 5), (ntok, heads, case["dim"]), "f32") * 1.5).to(TYPES[case["type"]]), k_cache=cache(6), v_cache=cache(7),
                qstart=_ints(np.concatenate([[0], np.cumsum(new)])), len=_ints(whole), table=_ints(table),
                lo=_ints(np.concatenate([v[0] for v in lim])) if case["docs"] else None,
                hi=_ints(np.concatenate([v[1] for v in lim])) if case["prefix"] else None,
                slopes=2.0 ** (-8.0 * torch.arange(1, heads + 1, dtype=torch.float32, device="cuda") / heads) if case["alibi"] else None,
                out=torch.zeros((ntok, heads, case["dim"]), dtype=TYPES[case["type"]], device="cuda"),
                lse=torch.zeros((ntok, heads), dtype=torch.float32, device="cuda"))


def prepare(case, seed):
    return dict(plan=_prepare_plan, rope=_prepare_rope, attn=_prepare_attn)[case["kind"]](case, seed)


# ---------------------------------------------------------------------------------------------------- plain forms
def _plain_plan(s):
    n, bs, dev = s["n"], s["bs"], s["ctx"].device
    ctx, add, table = s["ctx"].long(), s["add"].long(), s["table"].long()
    keep, cols = s["shared"] // bs, torch.arange(s["width"], device=dev)
    done = s["done"] != 0
    # finished sequences give their own blocks back, in order, behind the free ones
    given = done[:, None] & (cols >= keep) & (cols < ((ctx + bs - 1) // bs)[:, None])
    at = s["nfree"].long() + torch.cumsum(given.flatten().long(), 0) - 1
    free = torch.cat([s["free"].long(), torch.zeros(1, dtype=torch.long, device=dev)])
    free[torch.where(given.flatten(), at, s["nblocks"])] = table.flatten()
    nfree = s["nfree"].long() + given.sum()
    ctx = torch.where(done, ctx.clamp_max(s["shared"]), ctx)
    # the sequences that fit, in order
    held = (ctx + bs - 1) // bs
    need = torch.where(add > 0, (ctx + add + bs - 1) // bs - held, 0)
    fits = (torch.cumsum(need, 0) <= nfree) & (torch.cumsum(add, 0) <= s["ntok"]) & (ctx + add <= s["width"] * bs)
    fits = torch.cumprod(fits.long(), 0)
    add, need = add * fits, need * fits
    first = torch.cumsum(need, 0) - need
    new = (cols >= held[:, None]) & (cols < (held + need)[:, None])
    block = free[(nfree - 1 - (first[:, None] + cols - held[:, None])).clamp(0, s["nblocks"] - 1)]
    table = torch.where(new, block, table)
    qstart = torch.cat([torch.zeros(1, dtype=torch.long, device=dev), torch.cumsum(add, 0)])
    t = torch.arange(s["ntok"], device=dev)
    seq = torch.searchsorted(qstart[1:], t, right=True).clamp_max(n - 1)
    pos = ctx[seq] + t - qstart[seq]
    live = t < qstart[-1]
    slot = table[seq, (pos // bs).clamp_max(s["width"] - 1)] * bs + pos % bs
    i = lambda v: v.to(torch.int32)  # noqa: E731
    return dict(table=i(table), free=i(free[:-1]), nfree=i(nfree - need.sum()).reshape(1), len=i(ctx + add), qstart=i(qstart),
                pos=i(torch.where(live, pos, 0)), slot=i(torch.where(live, slot, -1)))


def _rotated(x, cos, sin, rot, inter):
    """x [n][heads][dim] in 32 bits; cos, sin [n][1][rot / 2]"""
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if inter else (x[..., :rot // 2], x[..., rot // 2:rot])
    u, v = a * cos - b * sin, b * cos + a * sin
    y = torch.stack([u, v], -1).flatten(-2) if inter else torch.cat([u, v], -1)
    return torch.cat([y, x[..., rot:]], -1)


def _plain_rope(s):
    h, kv = s["heads"], s["kv"]
    x = s["qkv"].float()
    angle = s["pos"].double()[:, None] * s["freq"]
    cos, sin = (angle.cos() * s["mag"]).float()[:, None], (angle.sin() * s["mag"]).float()[:, None]
    q = _rotated(x[:, :h], cos, sin, s["rot"], s["inter"])
    k = _rotated(x[:, h:h + kv], cos, sin, s["rot"], s["inter"])
    block, at = s["slot"].long() // s["bs"], s["slot"].long() % s["bs"]
    s["k_cache"][block, :, at] = k.to(s["k_cache"].dtype)
    s["v_cache"][block, :, at] = x[:, h + kv:].to(s["v_cache"].dtype)
    return dict(q=q.to(s["q"].dtype), k=s["k_cache"], v=s["v_cache"])


def _plain_attn(s):
    n, g, dim, maxq, dev = s["n"], s["heads"] // s["kv"], s["dim"], s["max_q"], s["q"].device
    start, whole, table = s["qstart"].long(), s["len"].long(), s["table"].long()
    keys = lambda c: c[table].float().permute(0, 2, 1, 3, 4).reshape(n, s["kv"], -1, dim)  # noqa: E731  [seq][head][position][dim]
    k, v = keys(s["k_cache"]), keys(s["v_cache"])
    # queries by sequence, padded to the longest
    j = torch.arange(maxq, device=dev)
    count = start[1:] - start[:-1]
    tok = (start[:-1, None] + j).clamp_max(s["ntok"] - 1)
    q = s["q"][tok].float().reshape(n, maxq, s["kv"], g, dim).permute(0, 2, 3, 1, 4).reshape(n, s["kv"], g * maxq, dim)
    pos = (whole - count)[:, None] + j                    # [seq][query]
    p = torch.arange(k.shape[2], device=dev)
    lo = torch.zeros_like(pos) if s["lo"] is None else s["lo"].long()[tok]
    hi = pos + 1 if s["hi"] is None else s["hi"].long()[tok]
    if s["window"]:
        lo = torch.maximum(lo, pos - s["window"])
    hi = torch.minimum(hi, whole[:, None])
    sees = (p >= lo[..., None]) & (p < hi[..., None])    # [seq][query][position]
    x = torch.matmul(q, k.transpose(2, 3).contiguous()).reshape(n, s["kv"], g, maxq, -1) * s["scale"]
    if s["cap"]:
        x = torch.tanh(x / s["cap"]) * s["cap"]
    if s["slopes"] is not None:
        x = x - s["slopes"].reshape(1, s["kv"], g, 1, 1) * (pos[..., None] - p).abs()[:, None, None]
    x = x.masked_fill_(~sees[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    x = (x - top).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.reshape(n, s["kv"], g * maxq, -1), v).reshape(n, s["kv"], g, maxq, dim) / total.clamp_min(1e-38)
    lse = (top + total.log()).squeeze(-1)
    # back to the batch's order of tokens
    t = torch.arange(s["ntok"], device=dev)
    seq = torch.searchsorted(start[1:], t, right=True)
    at = t - start[seq]
    o = o.permute(0, 3, 1, 2, 4).reshape(n, maxq, s["heads"], dim)[seq, at]
    return dict(out=o.to(s["out"].dtype), lse=lse.permute(0, 3, 1, 2).reshape(n, maxq, s["heads"])[seq, at])


# ---------------------------------------------------------------------------------------------------- the library
def _lib():
    if "maplemoe" not in sys.modules:
        sys.path.insert(0, os.path.join(ROOT, "maple-runtime_amd"))
    import maplemoe as M
    return M, M.lib()


def _p(t):
    return None if t is None else t.data_ptr()


def _cache(M, s):
    return M.KvCache(k=_p(s["k_cache"]), v=_p(s["v_cache"]), block_stride=s["kv"] * s["bs"] * s["dim"], head_stride=s["bs"] * s["dim"],
                     token_stride=s["dim"], nblocks=s["k_cache"].shape[0], block_size=s["bs"], heads=s["kv"], head_dim=s["dim"],
                     dtype=M.DTYPE[s.get("tout") or s["type"]])


def _own_plan(s):
    M, lib = _lib()
    a = M.KvPlan(ctx=_p(s["ctx"]), add=_p(s["add"]), done=_p(s["done"]), table=_p(s["table"]), free_list=_p(s["free"]), nfree=_p(s["nfree"]),
                 nfree_out=_p(s["nfree_out"]), len=_p(s["len"]), qstart=_p(s["qstart"]), pos=_p(s["pos"]), slot=_p(s["slot"]), nseq=s["n"],
                 width=s["width"], nblocks=s["nblocks"], block_size=s["bs"], shared=s["shared"], ntok=s["ntok"])
    M.check(lib.mmoe_kv_plan(a), "mmoe_kv_plan")
    return dict(table=s["table"], free=s["free"], nfree=s["nfree_out"], len=s["len"], qstart=s["qstart"], pos=s["pos"], slot=s["slot"])


def _own_rope(s):
    M, lib = _lib()
    h, kv, dim, row = s["heads"], s["kv"], s["dim"], s["qkv"].stride(0)
    x, size = s["qkv"].data_ptr(), s["qkv"].element_size()
    a = M.Rope(q=x, k=x + h * dim * size, v=x + (h + kv) * dim * size, q_out=_p(s["q"]), q_token=row, q_head=dim, k_token=row, k_head=dim, v_token=row,
               v_head=dim, qo_token=h * dim, qo_head=dim, pos=_p(s["pos"]), slot=_p(s["slot"]), freq=_p(s["freq"]), ntok=s["n"], heads=h, kv_heads=kv,
               head_dim=dim, rot=s["rot"], interleaved=int(s["inter"]), in_dtype=M.DTYPE[s["tin"]], out_dtype=M.DTYPE[s["tout"]], mag=s["mag"])
    M.check(lib.mmoe_rope_kv(a, _cache(M, s)), "mmoe_rope_kv")
    return dict(q=s["q"], k=s["k_cache"], v=s["v_cache"])


def _own_attn(s):
    M, lib = _lib()
    h, dim = s["heads"], s["dim"]
    a = M.PagedAttn(q=_p(s["q"]), out=_p(s["out"]), lse=_p(s["lse"]), q_token=h * dim, q_head=dim, out_token=h * dim, out_head=dim,
                    qstart=_p(s["qstart"]), len=_p(s["len"]), table=_p(s["table"]), lo=_p(s["lo"]), hi=_p(s["hi"]), slopes=_p(s["slopes"]), nseq=s["n"],
                    ntok=s["ntok"], heads=h, width=s["width"], max_q=s["max_q"], max_len=s["max_len"], shared=s["shared"], window=s["window"],
                    scale=s["scale"], cap=s["cap"])
    c = _cache(M, s)
    if "ws" not in s:   # a program keeps one for all its calls
        s["ws"] = torch.empty(lib.mmoe_attn_paged_ws(a, c), dtype=torch.uint8, device="cuda")
    a.ws, a.ws_bytes = s["ws"].data_ptr(), s["ws"].numel()
    M.check(lib.mmoe_attn_paged(a, c), "mmoe_attn_paged")
    return dict(out=s["out"], lse=s["lse"])


def run(state):
    if own:
        return dict(plan=_own_plan, rope=_own_rope, attn=_own_attn)[state["kind"]](state)
    return dict(plan=_plain_plan, rope=_plain_rope, attn=_plain_attn)[state["kind"]](state)


# ---------------------------------------------------------------------------------------------------- work
def work(case):
    if case["kind"] == "plan":
        ctx, add = _lens(case)
        bs = case["bs"]
        need = sum(_up(c + a, bs) - _up(c, bs) for c, a in zip(ctx, add)) * (0.7 if case["tight"] else 1.0)
        back = sum(_up(c, bs) - case["shared"] // bs for c in ctx[:case["done"]])
        # lengths, flags and last blocks in, lengths and starts out; blocks given back and taken; positions and slots
        return dict(bytes=4.0 * (6 * case["nseq"] + 2 * need + 2 * back + 2 * (sum(add) + case["pad"])), flops=0.0)
    if case["kind"] == "rope":
        e = lambda t: 4 if t == "f32" else 2  # noqa: E731
        vals = case["n"] * (case["heads"] + 2 * case["kv"]) * case["dim"]
        return dict(bytes=vals * (e(case["tin"]) + e(case["tout"])) + 8.0 * case["n"],
                    flops=3.0 * case["n"] * (case["heads"] + case["kv"]) * case["rot"])
    pairs, keys = 0, case["shared"]
    new, whole = _seqs(case)
    for q, n in zip(new, whole):
        lo, hi = _limits(case, q, n)
        if case["window"]:
            lo = np.maximum(lo, np.arange(n - q, n) - case["window"])
        pairs += int((hi - lo).sum())
        keys += int(hi.max() - max(int(lo.min()), case["shared"]))
    rows = sum(new) * case["heads"]
    return dict(bytes=rows * (case["dim"] * 4.0 + 4) + keys * case["kv"] * case["dim"] * 4.0, flops=4.0 * case["dim"] * case["heads"] * pairs)


# ---------------------------------------------------------------------------------------------------- in 64 bits
def _exact_rope(s):
    """rotation as a product of complex numbers; the caches written token by token through flat indexes"""
    h, kv, rot, bs = s["heads"], s["kv"], s["rot"], s["bs"]
    x = s["qkv"].double()
    turn = torch.polar(torch.full_like(s["freq"], s["mag"])[None].expand(s["n"], -1).contiguous(), torch.outer(s["pos"].double(), s["freq"]))[:, None]
    i = torch.arange(rot // 2, device=x.device)
    a, b = (2 * i, 2 * i + 1) if s["inter"] else (i, i + rot // 2)
    z = torch.complex(x[:, :h + kv][..., a], x[:, :h + kv][..., b]) * turn
    y = x.clone()
    y[:, :h + kv, a], y[:, :h + kv, b] = z.real, z.imag
    caches = []
    for c, new in ((s["k_cache"], y[:, h:h + kv]), (s["v_cache"], y[:, h + kv:])):
        c = c.double().transpose(1, 2).reshape(-1, kv, s["dim"]).index_copy(0, s["slot"].long(), new)
        caches.append(c.reshape(-1, bs, kv, s["dim"]).transpose(1, 2).contiguous())
    return dict(q=y[:, :h].contiguous(), k=caches[0], v=caches[1])


def _exact_attn(case, s):
    """sequence by sequence and head by head"""
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["lse"].shape, -math.inf, dtype=torch.float64, device="cuda")
    start, whole, g = s["qstart"].tolist(), s["len"].tolist(), s["heads"] // s["kv"]
    for b in range(s["n"]):
        t0, t1, n = start[b], start[b + 1], whole[b]
        q = t1 - t0
        rows = s["table"][b, :_up(n, s["bs"])].long()
        lo, hi = (torch.from_numpy(v).cuda() for v in _limits(case, q, n))
        pos, p = torch.arange(n - q, n, device="cuda"), torch.arange(n, device="cuda")
        hidden = (p < lo[:, None]) | (p >= hi[:, None])
        if s["window"]:
            hidden |= p < pos[:, None] - s["window"]
        far = (pos[:, None] - p).abs().double()
        for c in range(s["kv"]):
            k = s["k_cache"][rows, c].reshape(-1, s["dim"])[:n].double()
            v = s["v_cache"][rows, c].reshape(-1, s["dim"])[:n].double()
            for h in range(c * g, c * g + g):
                x = (s["q"][t0:t1, h].double() @ k.t().contiguous()) / math.sqrt(s["dim"])
                if s["cap"]:
                    x = s["cap"] * torch.tanh(x / s["cap"])
                if s["slopes"] is not None:
                    x = x - s["slopes"][h].double() * far
                x = x.masked_fill(hidden, -math.inf)
                lse[t0:t1, h] = torch.logsumexp(x, 1)
                out[t0:t1, h] = torch.softmax(x, 1) @ v
    return dict(out=out, lse=lse)


def exact(case, seed):
    if case["kind"] == "plan":
        return None   # whole numbers
    s = prepare(case, seed)
    return _exact_rope(s) if case["kind"] == "rope" else _exact_attn(case, s)
