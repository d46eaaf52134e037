"""Kernels that keep to their registers. What does not fit is kept in memory that the runtime sets aside for every lane that the chip can hold, and does not give back: 604 bytes
a lane were 320 MB. Read from what the compiler notes beside the kernels of the built library."""
import os
import re
import struct
import subprocess

import pytest

import thundergbm_amd as T
from thundergbm_amd import _lib

READELF = "/opt/rocm/llvm/bin/llvm-readelf"
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def code_objects(path):
    """The GPU's parts of a library: bundles of (offset, size, name) entries."""
    with open(path, "rb") as f:
        data = f.read()
    at = data.find(MAGIC)
    while at >= 0:
        place, (entries,) = at + len(MAGIC) + 8, struct.unpack_from("<Q", data, at + len(MAGIC))
        for _ in range(entries):
            offset, size, length = struct.unpack_from("<QQQ", data, place)
            name = data[place + 24:place + 24 + length]
            place += 24 + length
            if b"gfx950" in name and size:
                yield data[at + offset:at + offset + size]
        at = data.find(MAGIC, at + 1)


@pytest.fixture(scope="module")
def scratch(tmp_path_factory):
    """Bytes a lane of every kernel, by its mangled name."""
    T.load()
    if not os.path.exists(READELF):
        pytest.skip("no llvm-readelf")
    out, path = {}, str(tmp_path_factory.mktemp("code") / "part.o")
    for part in code_objects(_lib.LIB_PATH):
        with open(path, "wb") as f:
            f.write(part)
        notes = subprocess.run([READELF, "--notes", path], capture_output=True, text=True, check=True).stdout
        for kernel in notes.split("- .agpr_count:")[1:]:
            name, size = re.search(r"\.name: +(\S+)", kernel), re.search(r"\.private_segment_fixed_size: +(\d+)", kernel)
            out[name.group(1)] = int(size.group(1))
    return out


def test_kernels_of_the_product(scratch):
    names = [n for n in scratch if re.search(r"\d+k_(linear_few|linear_tiles|quantise|quantise_long|pack)I?", n)]
    assert len(names) > 40
    assert {n: scratch[n] for n in names if scratch[n]} == {}
