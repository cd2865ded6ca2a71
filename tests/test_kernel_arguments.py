"""How much the kernels of many sequences are passed, from the built library's own notes (no GPU needed)."""
import maplemoe as M

RUNTIME = 256   # bytes that the compiler adds behind a kernel's own arguments


def arguments():
    """kernel -> bytes of arguments (msgpack: a map's keys are sorted, so the size comes before the name)"""
    blob, out, at = open(M.LIB_PATH, "rb").read(), {}, 0
    key, name = b".kernarg_segment_size", b".name"
    while (at := blob.find(key, at)) >= 0:
        at += len(key)
        c = blob[at]
        n = c if c < 0x80 else int.from_bytes(blob[at + 1:at + 1 + (1 << c - 0xcc)], "big")
        at = blob.find(name, at) + len(name)
        c = blob[at]
        size, at = (c & 31, at + 1) if c < 0xc0 else (blob[at + 1], at + 2) if c == 0xd9 else (int.from_bytes(blob[at + 1:at + 3], "big"), at + 3)
        out[blob[at:at + size].decode()] = n
    return out


def test_plain_attention_is_not_passed_what_drafted_tokens_need():
    """a launch waits for its arguments: with those of mmoe_attn_tree behind its own, mmoe_attn_paged took 13.7 us instead of 13.1 for 7 tokens"""
    got = arguments()
    plain = {k: n for k, n in got.items() if any(f in k for f in ("k_attn_few", "k_attn_tile", "k_attn_join"))}
    drafted = [n for k, n in got.items() if "k_attn_tree" in k]
    assert len(plain) == 36 and len(drafted) == 32
    assert max(plain.values()) <= RUNTIME + 416 + 8 < min(drafted), plain
