"""What the compiler made of the latent kernels, read from the built library: no GPU is needed.

A fragment of four registers of which the compiler put three into scratch memory and one into an
accumulator register came back without the fourth (the kernel for gathered weights with 17 to 32 query
rows gave NaN): no latent kernel keeps registers in scratch memory."""
import os
import re
import struct
import subprocess

import pytest

from atomic_ops import _lib

LLVM = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin")


def _code_objects():
    """The gfx950 code objects that the library holds."""
    with open(_lib.LIB_PATH, "rb") as f:
        data = f.read()
    for m in re.finditer(b"__CLANG_OFFLOAD_BUNDLE__", data):
        at, p = m.start(), m.start() + 32
        for _ in range(struct.unpack_from("<Q", data, at + 24)[0]):
            off, size, name = struct.unpack_from("<QQQ", data, p)
            if size and b"gfx950" in data[p + 24:p + 24 + name]:
                yield data[at + off:at + off + size]
            p += 24 + name


def _tool(name, *args):
    exe = os.path.join(LLVM, name)
    if not os.path.exists(exe):
        pytest.skip(f"{name} not available")
    return subprocess.run([exe, *args], check=True, capture_output=True, text=True).stdout


@pytest.fixture(scope="module")
def latent_objects(tmp_path_factory):
    """(path, notes) of the code objects with latent kernels."""
    found = []
    for i, code in enumerate(_code_objects()):
        path = tmp_path_factory.mktemp("code") / f"{i}.elf"
        path.write_bytes(code)
        notes = _tool("llvm-readelf", "--notes", str(path))
        if re.search(r"\.name:\s+\S*(latent|evict)_", notes):
            found.append((str(path), notes))
    assert found
    return found


def test_no_registers_in_scratch_memory(latent_objects):
    seen = 0
    for _, notes in latent_objects:
        for kernel in notes.split("- .agpr_count:")[1:]:
            name = re.search(r"\.name:\s+(\S+)", kernel)[1]
            get = lambda key: int(re.search(rf"\.{key}:\s+(\d+)", kernel)[1])  # noqa: B023,E731
            assert get("vgpr_spill_count") == get("private_segment_fixed_size") == 0, name
            seen += 1
    assert seen > 50
