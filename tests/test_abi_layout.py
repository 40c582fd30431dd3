"""The C structures of ABI version 2 keep their layout: a program built against an earlier header of that version passes them as they were."""
import ctypes as C


def _fields(spec):
    """(size, alignment) of each field of "i4 i4 l8 p8", as C lays them out."""
    return [(int(f[1:]), int(f[1:])) for f in spec.split()]


def _size(spec):
    at = 0
    for size, align in _fields(spec):
        at = -(-at // align) * align + size
    most = max(a for _, a in _fields(spec))
    return -(-at // most) * most


def test_a_decoding_step_takes_the_descriptor_of_earlier_headers():
    from memory_b200 import _lib as L
    assert L.lib().moc_abi_version() == 2
    assert C.sizeof(L.RouterShape) == _size("i4 " * 6 + "f4 i4") and C.sizeof(L.DecodeShape) == _size("i4 " * 7 + "f4")
    # router, attn, hidden_dtype, out_dim, bank_rows, 16 pointers, hidden_dim, launches: the last field ends the structure
    words = C.sizeof(L.RouterShape) + C.sizeof(L.DecodeShape)
    assert C.sizeof(L.DecodeStepDesc) == words + 2 * 4 + 8 + 16 * 8 + 2 * 4
    assert L.DecodeStepDesc.launches.offset + 4 == C.sizeof(L.DecodeStepDesc)


def test_the_header_ends_the_descriptor_at_its_earlier_last_field():
    import os
    import re
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "moc_b200.h")).read()
    body = re.sub(r"/\*.*?\*/", "", text[:text.index("} moc_decode_step_desc;")].rsplit("typedef struct {", 1)[1], flags=re.S)
    assert body.split()[-2:] == ["int32_t", "launches;"]


def test_the_clipping_workspace_grows_with_every_table():
    """A launch holds 64 tensors, or 680: one more asks for the partial sums of another launch."""
    from memory_b200 import _lib as L
    size = L.lib().moc_grad_clip_workspace_bytes
    assert size(0) == size(63) > 0 and size(65) == size(679)
    assert size(64 + 2 * 680) > size(64 + 680) > size(65) and size(680 * 3) > size(680 * 2) > size(680 * 1 - 1)


def test_the_8_bit_step_refuses_without_a_gpu():
    from memory_b200 import _lib as L
    assert L.lib().moc_decode_step_cache(None, None, 0) == -1
    s = L.DecodeStepDesc()
    assert L.lib().moc_decode_step_cache(C.byref(s), 4096, 8) == -1 and L.lib().moc_decode_step(C.byref(s)) == -1
