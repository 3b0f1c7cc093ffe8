"""Registers of the built kernels, from the notes that the compiler leaves beside them in libkq.so: what
a kernel's waves a SIMD go by. On the CPU; nothing is run."""
import os
import re
import struct
import subprocess

import pytest

from kernels_amd import build, kq

READELF = os.path.join(build.ROCM, "llvm", "bin", "llvm-readelf")


def code_objects():
    """The gfx950 parts of the library's bundles."""
    kq.lib()  # raises if it was not built
    with open(build.LIB, "rb") as f:
        data = f.read()
    magic = b"__CLANG_OFFLOAD_BUNDLE__"
    at = data.find(magic)
    while at >= 0:
        p = at + len(magic) + 8
        for _ in range(struct.unpack_from("<Q", data, at + len(magic))[0]):
            off, size, name = struct.unpack_from("<QQQ", data, p)
            if size and build.ARCH.encode() in data[p + 24:p + 24 + name]:
                yield data[at + off:at + off + size]
            p += 24 + name
        at = data.find(magic, at + 1)


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """{mangled name: (registers of a lane, bytes of scratch)}"""
    got, path = {}, str(tmp_path_factory.mktemp("notes") / "object")
    for one in code_objects():
        with open(path, "wb") as f:
            f.write(one)
        notes = subprocess.run([READELF, "--notes", path], capture_output=True, text=True, check=True).stdout
        for kernel in notes.split("- .agpr_count:")[1:]:
            field = lambda key: re.search(rf"\.{key}:\s+(\S+)", kernel).group(1)  # noqa: E731
            got[field("name")] = int(field("vgpr_count")), int(field("private_segment_fixed_size"))
    return got


def waves(registers):
    """Of a SIMD's 512 registers, in eights."""
    return min(512 // (-(-registers // 8) * 8), 8)


@pytest.mark.parametrize("dim,least", [(64, 8), (96, 5), (128, 4), (192, 2), (256, 2)])
def test_waves_of_kv_write(kernels, dim, least):
    found = {n: r for n, r in kernels.items() if f"kv_write_kILi{dim}E" in n}
    assert len(found) == 4, "int8 and e4m3 codes, of fp16 and bf16"
    for name, (registers, scratch) in found.items():
        assert waves(registers) >= least and scratch == 0, (name, registers, scratch)
