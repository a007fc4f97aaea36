"""Registers of the built kernels, as the compiler wrote them into the library."""

from __future__ import annotations

import pathlib
import struct

import msgpack
import pytest

LIB = pathlib.Path(__file__).resolve().parents[1] / "myelin_amd" / "libmyelin_hip.so"
BUNDLE = b"__CLANG_OFFLOAD_BUNDLE__"


def _note(elf: bytes) -> bytes:
    """The code object's metadata: the AMDGPU note (type 32) of its ELF file."""

    shoff, = struct.unpack_from("<Q", elf, 0x28)
    shentsize, shnum = struct.unpack_from("<HH", elf, 0x3A)
    for i in range(shnum):
        _, kind, _, _, offset, size = struct.unpack_from("<IIQQQQ", elf, shoff + i * shentsize)
        if kind != 7:  # SHT_NOTE
            continue
        at = offset
        while at < offset + size:
            namesz, descsz, note = struct.unpack_from("<III", elf, at)
            desc = at + 12 + (namesz + 3) // 4 * 4
            if note == 32:
                return elf[desc : desc + descsz]
            at = desc + (descsz + 3) // 4 * 4
    raise AssertionError("no metadata")


@pytest.fixture(scope="module")
def kernels():
    if not LIB.exists():
        pytest.skip("libmyelin_hip.so is not built")
    data, found, at = LIB.read_bytes(), {}, 0
    while (at := data.find(BUNDLE, at)) >= 0:
        count, = struct.unpack_from("<Q", data, at + 24)
        entry = at + 32
        for _ in range(count):
            offset, size, length = struct.unpack_from("<QQQ", data, entry)
            target = data[entry + 24 : entry + 24 + length]
            entry += 24 + length
            if b"gfx950" in target and size:
                meta = msgpack.unpackb(_note(data[at + offset : at + offset + size]))
                found |= {k[".name"]: k for k in meta["amdhsa.kernels"]}
        at += len(BUNDLE)
    return found


def test_decay_attention_keeps_its_registers(kernels):
    """A spilled register is stored and loaded in every chunk: 114 of them cost fp32
    of 128 x 128 a third of its time.  The 8-wave bf16 kernels, which two
    workgroups a CU hold to 128 registers, are let off a few."""

    chunked = {n: k for n, k in kernels.items() if "chunked" in n}
    assert len(chunked) >= 20
    spilled = {n: k[".vgpr_spill_count"] for n, k in chunked.items() if k[".vgpr_spill_count"]}
    assert all("BF16ELi8ELi8E" in n and count <= 5 for n, count in spilled.items()), spilled
