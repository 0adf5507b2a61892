"""The registers of the norms' kernels in the built library, as its code objects state
them: rows of 8193 to 16384 columns take workgroups of 1024 threads, of which a compute
unit holds two only if a thread has 64 vector registers at most (4096 rows of 12288
quantised: 34 us so, 49 with one workgroup a unit)."""
import os
import re
import shutil
import struct
import subprocess

import pytest

from hachiue_amd import sampler as hs

READELF = shutil.which("llvm-readelf", path="/opt/rocm/llvm/bin:" + os.environ.get("PATH", ""))
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def code_objects():
    data = open(hs.LIB_PATH, "rb").read()
    at = data.find(MAGIC)
    while at >= 0:
        (count,), p = struct.unpack_from("<Q", data, at + len(MAGIC)), at + len(MAGIC) + 8
        for _ in range(count):
            offset, size, name = struct.unpack_from("<QQQ", data, p)
            target = data[p + 24:p + 24 + name].decode()
            p += 24 + name
            if "gfx950" in target and size:
                yield data[at + offset:at + offset + size]
        at = data.find(MAGIC, at + 1)


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """{name of a norm's kernel: (vector registers, spilled ones)}"""
    if not READELF:
        pytest.skip("llvm-readelf is not installed")
    path, found = tmp_path_factory.mktemp("code") / "object", {}
    for obj in code_objects():
        path.write_bytes(obj)
        notes = subprocess.run([READELF, "--notes", str(path)], capture_output=True, text=True, check=True).stdout
        for part in notes.split("- .agpr_count:")[1:]:
            name = re.search(r"\.name: +(\S+)", part).group(1)
            if m := re.search(r"block_norm_kernelILi(\d+)ELi(\d+)ELb(\d)E", name):
                found[tuple(map(int, m.groups()))] = tuple(
                    int(re.search(rf"\.{key}: +(\d+)", part).group(1)) for key in ("vgpr_count", "vgpr_spill_count"))
    return found


def test_every_form_is_there_and_spills_nothing(kernels):
    assert len(kernels) == 18
    assert all(spilled == 0 for _, spilled in kernels.values()), kernels


def test_two_workgroups_of_a_wide_row_fit_on_a_unit(kernels):
    registers, _ = kernels[2, 1024, 1]
    assert registers <= 64
