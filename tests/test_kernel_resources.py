"""What the compiler gave the built kernels (no GPU needed): read from the code
objects in librqmv.so."""
import struct

import pytest

import rqmv

msgpack = pytest.importorskip("msgpack")


def code_objects(data: bytes):
    """The gfx950 ELF images of every offload bundle in the library."""
    magic = b"__CLANG_OFFLOAD_BUNDLE__"
    at = data.find(magic)
    while at >= 0:
        count, = struct.unpack_from("<Q", data, at + 24)
        pos = at + 32
        for _ in range(count):
            offset, size, length = struct.unpack_from("<QQQ", data, pos)
            name = data[pos + 24:pos + 24 + length]
            pos += 24 + length
            if b"gfx950" in name and size:
                yield data[at + offset:at + offset + size]
        at = data.find(magic, at + 1)


def kernels(elf: bytes):
    """The kernels' metadata (the AMDGPU note of an ELF image)."""
    start, = struct.unpack_from("<Q", elf, 0x28)
    each, count = struct.unpack_from("<HH", elf, 0x3A)
    for i in range(count):
        _, kind, _, _, offset, size = struct.unpack_from("<IIQQQQ", elf, start + i * each)
        if kind != 7:  # SHT_NOTE
            continue
        pos = offset
        while pos < offset + size:
            name_size, desc_size, note = struct.unpack_from("<III", elf, pos)
            desc = pos + 12 + (name_size + 3) // 4 * 4
            if note == 32:  # NT_AMDGPU_METADATA
                yield from msgpack.unpackb(elf[desc:desc + desc_size])["amdhsa.kernels"]
            pos = desc + (desc_size + 3) // 4 * 4


@pytest.fixture(scope="module")
def built():
    with open(rqmv.LIB_PATH, "rb") as f:
        found = {k[".name"]: k for elf in code_objects(f.read()) for k in kernels(elf)}
    assert len(found) > 100
    return found


@pytest.mark.parametrize("name", ["paged_few_kernel", "paged_many_kernel", "paged_join_kernel", "paged_items_kernel"])
def test_attention_over_pages_spills_no_registers(built, name):
    """A reload inside the key loop waits for the step's own loads to LDS, which the compiler does not count."""
    mine = {n: k for n, k in built.items() if name in n}
    assert len(mine) == {"paged_few_kernel": 6, "paged_many_kernel": 6, "paged_join_kernel": 18}.get(name, 1)
    for n, k in mine.items():
        assert k[".private_segment_fixed_size"] == 0 and k[".vgpr_spill_count"] == 0, n
