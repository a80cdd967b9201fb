"""How the sequence-block sources are built, and what the compiler made of the fp8 product: its matrix instructions stand in inline assembly, where the compiler knows neither that a result
takes its passes to arrive nor that it may not be looked at before.  Read from the built library."""
import os
import re
import runpy
import struct
import subprocess
import sys

import pytest

from tecogan_amd import _lib as L
from tecogan_amd import build as B

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


@pytest.mark.parametrize("src", B.SOURCES)
def test_a_variant_of_a_source_is_built_with_that_sources_flags(src, monkeypatch):
    """tools/build_variant.py against the build itself: an A/B of the two compares nothing but what -D changes."""
    calls, tool = [], os.path.join(os.path.dirname(B.HERE), "tools", "build_variant.py")
    monkeypatch.setattr(subprocess, "check_call", lambda cmd, **kw: calls.append(cmd))
    monkeypatch.setattr(B, "build", lambda **kw: None)
    monkeypatch.setattr(sys, "argv", [tool, src, "-DX=1"])
    runpy.run_path(tool)
    assert calls[0][1:-5] == B.flags_for(src) and calls[0][-5] == "-DX=1"
    assert ("-packed-fp32-ops" in calls[0]) == (src in B.SCALAR_FP32_SOURCES)


def code_objects(path):
    """The gfx950 code objects of a library: each compiled source's bundle has a magic, a count, and (offset, size, name) of its entries."""
    data = open(path, "rb").read()
    for m in re.finditer(b"__CLANG_OFFLOAD_BUNDLE__", data):
        n, = struct.unpack_from("<Q", data, m.end())
        at = m.end() + 8
        for _ in range(n if n < 16 else 0):
            offset, size, length = struct.unpack_from("<QQQ", data, at)
            name = data[at + 24:at + 24 + length]
            at += 24 + length
            if b"gfx950" in name:
                yield data[m.start() + offset:m.start() + offset + size]


@pytest.fixture(scope="module")
def tile_kernels(tmp_path_factory):
    """Instructions of every fp8_tile_kernel, by name."""
    L.lib()                                          # builds nothing, but says so where there is no library
    own = [c for c in code_objects(L.LIB_PATH) if b"fp8_tile_kernel" in c]
    assert len(own) == 1
    path = os.path.join(str(tmp_path_factory.mktemp("code")), "fp8.co")
    open(path, "wb").write(own[0])
    kernels, now = {}, None
    for line in subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", path], check=True, capture_output=True, text=True).stdout.splitlines():
        head = re.match(r"^[0-9a-f]+ <(.*)>:", line)
        if head:
            now = kernels.setdefault(head.group(1), []) if "fp8_tile_kernel" in head.group(1) else None
        elif now is not None and line.startswith("\t"):
            now.append(line.split("//")[0].strip())
    return kernels


def registers(text):
    out = set()
    for one, lo, hi in re.findall(r"\ba(?:(\d+)|\[(\d+):(\d+)\])", text):
        out |= {int(one)} if one else set(range(int(lo), int(hi) + 1))
    return out


def test_nobody_touches_an_accumulator_between_the_matrix_instructions(tile_kernels):
    assert len(tile_kernels) >= 20                   # formats x sums x tiles
    for name, code in tile_kernels.items():
        at = [i for i, s in enumerate(code) if s.startswith("v_mfma")]
        sums = set().union(*(registers(code[i].split(",")[0]) for i in at))
        assert len(sums) in (16, 64, 256), name      # 4 x fragments, no second set
        for s in code[at[0]:at[-1]]:
            assert s.startswith("v_mfma") or not registers(s) & sums, (name, s)
        waits = 0                                    # a result is there 18 states behind the longest instruction
        for s in code[at[-1] + 1:]:
            if registers(s) & sums:
                break
            waits += int(s.split()[1]) + 1 if s.startswith("s_nop") else 1
        assert waits >= 18, (name, waits)


def test_tiles_spill_nothing(tile_kernels):
    """A spilled accumulator would be stored before it is there."""
    for name, code in tile_kernels.items():
        assert not [s for s in code if s.startswith("scratch_")], name
