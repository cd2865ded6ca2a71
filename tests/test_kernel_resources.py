"""What the compiler made of the kernels, from the built library's own notes (no GPU needed)."""
import maplemoe as M


def notes(field):
    """a number of every kernel, in the order of the code objects"""
    blob, key, out, at = open(M.LIB_PATH, "rb").read(), b"." + field.encode(), [], 0
    while (at := blob.find(key, at)) >= 0:
        at += len(key)
        if blob[at] < 0x80:
            out.append(blob[at])
        elif blob[at] in (0xcc, 0xcd, 0xce):      # msgpack: an unsigned number of 1, 2 or 4 bytes
            out.append(int.from_bytes(blob[at + 1:at + 1 + (1 << blob[at] - 0xcc)], "big"))
    return out


def test_no_kernel_of_many_sequences_spills_vector_registers():
    """A vector register that this compiler spills behind a branch taken by some lanes only is stored for those lanes alone, where scalar registers are
    spilled at the same place: kernels that hold asm loads and so many registers must fit. One form of the experts' k_gateup_pk
    spills a few; nothing there branches by lane."""
    spills = notes("vgpr_spill_count")
    assert len(spills) > 150
    assert sum(x > 0 for x in spills) <= 1 and max(spills) <= 5, spills
