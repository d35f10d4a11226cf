"""What the compiler made of the kernels: read from the notes of the code objects in the built library."""
import os
import re
import struct
import subprocess

import pytest

from vllm_trianglemix_amd import _lib

READELF = "/opt/rocm/llvm/bin/llvm-readelf"


def code_objects(path):
    """The gfx950 code objects of a HIP library: every offload bundle is a magic word, a count, and (offset, size, name)
    entries."""
    data, magic = open(path, "rb").read(), b"__CLANG_OFFLOAD_BUNDLE__"
    at = data.find(magic)
    while at >= 0:
        n, pos = struct.unpack_from("<Q", data, at + len(magic))[0], at + len(magic) + 8
        for _ in range(n if n < 64 else 0):
            offset, size, chars = struct.unpack_from("<QQQ", data, pos)
            name = data[pos + 24:pos + 24 + chars]
            pos += 24 + chars
            if b"gfx950" in name and size:
                yield data[at + offset:at + offset + size]
        at = data.find(magic, at + 1)


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """Kernel -> (registers spilled, bytes of scratch a lane)."""
    if not os.path.exists(READELF):
        pytest.skip("no llvm-readelf")
    found, f = {}, tmp_path_factory.mktemp("objects") / "o"
    for obj in code_objects(_lib.LIB_PATH):
        f.write_bytes(obj)
        notes = subprocess.run([READELF, "--notes", str(f)], capture_output=True, text=True, check=True).stdout
        for part in notes.split("- .agpr_count:")[1:]:
            get = lambda key: int(re.search(key + r":\s+(\d+)", part).group(1))  # noqa: E731
            found[re.search(r"\.name:\s+(\S+)", part).group(1)] = get(r"\.vgpr_spill_count"), get(r"\.private_segment_fixed_size")
    return found


@pytest.mark.parametrize("kernel, forms", [("fp4_decode_kernel", 12), ("fp4_join_kernel", 12), ("fp4_write_kernel", 2), ("fp4_gather_kernel", 2),
                                           ("pg_copy_kernel", 4), ("pg_fork_kernel", 2), ("pg_small_kernel", 2)])
def test_no_registers_in_scratch(kernels, kernel, forms):
    """(A spilled register turns into memory accesses whose waits the loads in flight take part in.)"""
    mine = {k: v for k, v in kernels.items() if kernel in k}
    assert len(mine) == forms and all(v == (0, 0) for v in mine.values()), mine
