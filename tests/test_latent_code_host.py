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


def _sgprs(operand):
    m = re.fullmatch(r"s\[(\d+):(\d+)\]|s(\d+)", operand)
    if not m:
        return set()
    return {int(m[3])} if m[3] else set(range(int(m[1]), int(m[2]) + 1))


def test_scalar_addresses_are_there_when_a_load_reads_them(latent_objects):
    """A memory instruction may read a scalar register five wait states after a vector instruction has written
    it, and nothing in the card waits for that.  The compiler does not look into inline assembly, so what
    stands there has to wait by itself."""
    loads = 0
    for path, _ in latent_objects:
        wrote = {}                                  # scalar register: wait states since a vector instruction wrote it
        for line in _tool("llvm-objdump", "-d", path).splitlines():
            if line.endswith(">:"):
                wrote, where = {}, line
                continue
            op, _, rest = line.split("//")[0].strip().partition(" ")
            if not re.match(r"[vs]_|ds_|global_|buffer_|scratch_|flat_", op):
                continue
            operands = [x.strip() for x in re.split(r",|\s(?!\s)", rest) if x.strip()]
            if op.startswith(("global_", "buffer_", "scratch_", "flat_")):
                loads += 1
                for x in operands:
                    assert not _sgprs(x) & wrote.keys(), (where, line)
            states = int(operands[0]) + 1 if op == "s_nop" else 1
            wrote = {r: n + states for r, n in wrote.items() if n + states < 5}
            if op.startswith("v_"):
                wrote.update((r, 0) for x in operands[:2 if "_co_" in op or "div_scale" in op else 1] for r in _sgprs(x))
            elif op.startswith("s_") and operands:
                for r in _sgprs(operands[0]):
                    wrote.pop(r, None)
    assert loads > 1000
