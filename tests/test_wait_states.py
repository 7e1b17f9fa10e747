"""The built library's gfx950 code, disassembled: direct-to-LDS loads are written in inline assembly, in
which the compiler adds no wait states. A load of that kind needs one behind the scalar write of M0, which
holds its LDS address, and, as every load, five behind a vector instruction that wrote a scalar register it
reads (a value made uniform, or one brought back from where registers had run out)."""
from __future__ import annotations

import re
import shutil
import struct
import subprocess
from functools import lru_cache
from pathlib import Path

import pytest

from xkernels_amd import _lib, build

MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def _objdump() -> str:
    for cand in (Path(build.hipcc()).resolve().parent / "../llvm/bin/llvm-objdump", shutil.which("llvm-objdump"),
                 "/opt/rocm/llvm/bin/llvm-objdump"):
        if cand and Path(cand).exists():
            return str(cand)
    pytest.skip("no llvm-objdump")


def _code_objects(data: bytes):
    """The gfx950 code objects of the bundles in ``data``."""
    at = data.find(MAGIC)
    while at >= 0:
        n, = struct.unpack_from("<Q", data, at + len(MAGIC))
        p = at + len(MAGIC) + 8
        for _ in range(n):
            off, size, length = struct.unpack_from("<QQQ", data, p)
            name = data[p + 24:p + 24 + length]
            p += 24 + length
            if build.ARCH.encode() in name and size:
                yield data[at + off:at + off + size]
        at = data.find(MAGIC, p)


@lru_cache(maxsize=1)
def _loads():
    """For each direct-to-LDS load its text and the eight instructions before it, the nearest last."""
    import tempfile

    found = []
    with tempfile.TemporaryDirectory() as d:
        for i, code in enumerate(_code_objects(Path(_lib.LIB_PATH).read_bytes())):
            path = Path(d) / f"{i}.o"
            path.write_bytes(code)
            text = subprocess.run([_objdump(), "-d", "--no-show-raw-insn", str(path)], capture_output=True, text=True,
                                  check=True).stdout
            before: list[str] = []
            for line in text.splitlines():
                if not line.startswith("\t"):
                    before = []
                    continue
                line = line.split("//")[0].strip()
                if re.search(r"^(buffer|global)_load.*\blds\b", line):
                    found.append((line, tuple(before)))
                before = [*before[-7:], line]
    return found


def _states(line: str) -> int:
    """The wait states an instruction takes."""
    return int(line.split()[1], 0) + 1 if line.startswith("s_nop") else 1


def _since(before, writes) -> int:
    """Wait states between the nearest instruction that ``writes`` and the load."""
    n = 0
    for line in reversed(before):
        if writes(line):
            return n
        n += _states(line)
    return n


def test_wait_states_behind_m0():
    loads = _loads()
    assert loads
    bad = [(a, b[-1]) for a, b in loads if _since(b, lambda line: re.match(r"s_\w+ m0,", line)) < 1]
    assert not bad, f"{len(bad)} of {len(loads)} loads directly behind a write of M0, the first: {bad[0]}"


def _scalars(text: str) -> set[str]:
    """The scalar registers that operands name."""
    found = {"vcc"} if "vcc" in text else set()
    for first, last, one in re.findall(r"\bs\[(\d+):(\d+)\]|\bs(\d+)\b", text):
        found |= {f"s{n}" for n in (range(int(first), int(last) + 1) if first else (int(one),))}
    return found


def _written_by_vector(line: str) -> set[str]:
    """The scalar registers that a vector instruction writes (its first or, of a carry, second operand)."""
    name, _, operands = line.partition(" ")
    if not name.startswith("v_"):
        return set()
    return _scalars(",".join(operands.split(",")[:2 if "_co_" in name or "div_scale" in name else 1]))


def test_wait_states_behind_scalars_of_vector_instructions():
    loads = _loads()
    bad = [(a, b) for a, b in loads if _since(b, lambda line: _written_by_vector(line) & _scalars(a)) < 5]
    assert not bad, f"{len(bad)} of {len(loads)} loads, the first: {bad[0]}"
