"""What the compiler made of the paged attention kernels, read from the notes of
the library that was built here."""

import struct

import pytest

from mlx_batch_invariant import _lib

msgpack = pytest.importorskip("msgpack")


def _device_images(blob):
    """The gfx950 code objects of every offload bundle in a host library."""
    magic = b"__CLANG_OFFLOAD_BUNDLE__"
    at = blob.find(magic)
    while at >= 0:
        (count,) = struct.unpack_from("<Q", blob, at + 24)
        p = at + 32
        for _ in range(count):
            off, size, n = struct.unpack_from("<QQQ", blob, p)
            if size and b"gfx950" in blob[p + 24:p + 24 + n]:
                yield blob[at + off:at + off + size]
            p += 24 + n
        at = blob.find(magic, at + 24)


def _notes(elf):
    """The kernels' metadata of one code object (ELF note 32 of "AMDGPU")."""
    (phoff,) = struct.unpack_from("<Q", elf, 32)
    phsize, phnum = struct.unpack_from("<HH", elf, 54)
    for i in range(phnum):
        kind, _, off, _, _, size = struct.unpack_from("<IIQQQQ", elf, phoff + i * phsize)
        if kind != 4:  # PT_NOTE
            continue
        end = off + size
        while off < end:
            nlen, dlen, t = struct.unpack_from("<III", elf, off)
            name = elf[off + 12:off + 12 + nlen].rstrip(b"\0")
            data = off + 12 + (nlen + 3) // 4 * 4
            if name == b"AMDGPU" and t == 32:
                yield from msgpack.unpackb(elf[data:data + dlen])["amdhsa.kernels"]
            off = data + (dlen + 3) // 4 * 4


def paged_kernels():
    _lib.lib()  # builds nothing: fails if there is no library
    with open(_lib.LIB_PATH, "rb") as f:
        blob = f.read()
    return [k for image in _device_images(blob) for k in _notes(image) if "bi_paged" in k[".name"]]


def test_paged_attention_keeps_its_registers():
    """No paged attention kernel keeps vector registers in scratch memory."""
    kernels = paged_kernels()
    assert len(kernels) >= 6 * 3 * 4  # head dims, types, two split kernels, the fold and a whole one
    spilled = {k[".name"]: k[".vgpr_spill_count"] for k in kernels if k[".vgpr_spill_count"]}
    assert not spilled
