"""The early fetch of a kernel's arguments (include/mi355_kernels/kernarg.h) in the kernels as they were compiled, without a device: none of
its loads ends past the block of arguments that the kernel's launch has."""
import os
import re
import struct
import subprocess

import pytest

from attention_superoptimizer_amd import build as B

TOOLS = "/opt/rocm/llvm/bin"
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def _code_objects():
    """Those for gfx950 in the backend's library."""
    with open(B.BACKEND_LIB, "rb") as f:
        blob = f.read()
    at = blob.find(MAGIC)
    while at >= 0:
        count, place = struct.unpack_from("<Q", blob, at + len(MAGIC))[0], at + len(MAGIC) + 8
        for _ in range(count if count <= 8 else 0):  # (the name of the format alone is no bundle)
            offset, size, length = struct.unpack_from("<QQQ", blob, place)
            if b"gfx950" in blob[place + 24:place + 24 + length] and size > 0:
                yield blob[at + offset:at + offset + size]
            place += 24 + length
        at = blob.find(MAGIC, at + 1)


def _run(tool, *args):
    return subprocess.run([os.path.join(TOOLS, tool), *args], capture_output=True, check=True).stdout


def test_no_fetch_ends_past_the_arguments(tmp_path):
    if not os.path.exists(os.path.join(TOOLS, "llvm-objdump")):
        pytest.skip("no disassembler")
    fetch = re.compile(rb"(?:\ts_load_dword (s\d+), (s\[\d+:\d+\]), (0x[0-9a-f]+)[^\n]*\n)(?:\ts_load_dword \1, \2, 0x[0-9a-f]+[^\n]*\n){8}")
    kernel = re.compile(rb"^[0-9a-f]+ <(\w+)>:\n", re.M)
    fetching, past = [], []
    for i, code in enumerate(_code_objects()):
        path = tmp_path / f"{i}.co"
        path.write_bytes(code)
        notes = _run("llvm-readelf", "--notes", str(path)).decode()
        size_of = {name: int(size) for size, name in re.findall(r"\.kernarg_segment_size: (\d+)\n.*?\.name: +(\w+)\n", notes, re.S)}
        text = _run("llvm-objdump", "-d", "--no-show-raw-insn", str(path))
        begins = list(kernel.finditer(text))
        for begin, end in zip(begins, [m.start() for m in begins[1:]] + [len(text)]):
            name = begin.group(1).decode()
            for m in fetch.finditer(text, begin.end(), end):
                last = max(int(x, 16) for x in re.findall(rb", (0x[0-9a-f]+)", m.group()))
                fetching.append(name)
                if last + 4 > size_of[name]:
                    past.append((name, last + 4, size_of[name]))
    for which in ("attention_blocks_kernel", "join_blocks_kernel", "paged_attention_kernel", "log_probabilities_kernel"):
        assert any(which in name for name in fetching), which
    assert not past, past
