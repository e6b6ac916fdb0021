"""What the build promises and the compiler does not check: hand-written instructions in the sources and in the built kernels."""
import glob
import os
import re
import shutil
import subprocess

import pytest

from gpt_amd import _lib as L

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "g.pt_amd", "csrc")
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


def asm_statements():
    for name in sorted(os.listdir(CSRC)):
        if name.endswith((".h", ".hip")):
            text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())
            for start in (m.start() for m in re.finditer(r"\basm\b", text)):
                depth, end = 0, text.index("(", start)
                while True:                                              # to the matching parenthesis
                    depth += {"(": 1, ")": -1}.get(text[end], 0)
                    end += 1
                    if depth == 0:
                        break
                yield name, text[start:end]


def test_inline_assembly_declares_m0():
    """m0 is the compiler's as well (LDS-DMA builtins, indexed moves): a statement that sets it says so."""
    setters = [(name, text) for name, text in asm_statements() if re.search(r"\bm0, %", text)]
    assert len(setters) >= 2
    for name, text in setters:
        assert '"m0"' in text.rsplit(":", 1)[1], (name, text)


def scalars(operand):
    m = re.fullmatch(r"s\[(\d+):(\d+)\]|s(\d+)", operand)
    return set() if not m else {int(m[3])} if m[3] else set(range(int(m[1]), int(m[2]) + 1))


def hazards(lines):
    """LDS loads in a listing, and those whose scalar operands a vector instruction wrote fewer than five wait states before (branches are
    read past: a write on either way counts)."""
    loads, bad = 0, []
    recent = []                                                          # (scalars written by a vector instruction, wait states)
    for line in lines:
        op, _, rest = line.partition(" ")
        operands = [o.strip().split(" ")[0] for o in rest.split(",")]
        if op.startswith("buffer_load") and line.endswith("lds"):
            loads += 1
            read, states = set().union(*(scalars(o) for o in operands)), 0
            for written, n in reversed(recent):
                if written & read:
                    bad.append(line)
                    break
                states += n
                if states >= 5:
                    break
        n = int(operands[0], 0) + 1 if op == "s_nop" else 1
        recent = recent[-8:] + [(scalars(operands[0]) if op.startswith("v_") else set(), n)]
    return loads, bad


def test_hazards_are_seen():
    wrote, load = "v_readfirstlane_b32 s9, v1", "buffer_load_dwordx4 v2, s[8:11], 0 offen lds"
    assert hazards([wrote, "s_mov_b32 m0, s3", "s_nop 0", load]) == (1, [load])
    assert hazards([wrote, "s_nop 4", load]) == (1, []) and hazards([wrote] + ["v_mov_b32 v3, v4"] * 5 + [load]) == (1, [])
    assert hazards(["v_readfirstlane_b32 s12, v1", load, "s_mov_b32 s9, s1", load]) == (2, [])


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no disassembler")
def test_loads_to_lds_wait_for_their_descriptors(tmp_path):
    """The loads to LDS that are written out in assembly text: the compiler adds no wait states there."""
    library = shutil.copy(L.LIB_PATH, tmp_path)
    subprocess.run([OBJDUMP, "--offloading", library], cwd=tmp_path, check=True, stdout=subprocess.DEVNULL)
    loads = 0
    for code in glob.glob(os.path.join(tmp_path, "*amdgcn*")):
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "--no-leading-addr", code], check=True, capture_output=True, text=True).stdout
        n, bad = hazards([line.split("//")[0].strip() for line in text.splitlines() if line.startswith("\t")])
        loads += n
        assert not bad, (code, bad[:3])
    assert loads > 500


def included(name, seen=None):
    """The headers of this folder and the C interface that a source reads, through other headers too."""
    seen = set() if seen is None else seen
    for path in re.findall(r'#include "([^"]+)"', open(os.path.join(CSRC, name)).read()):
        if path not in seen:
            seen.add(path)
            included(path, seen)
    return seen


def would_build(*args):
    """The commands of a make that thinks these files have changed."""
    return subprocess.run(["make", "-n", "-C", CSRC, *args], check=True, capture_output=True, text=True).stdout


def test_a_changed_header_rebuilds_every_object_that_reads_it():
    sources = [n for n in os.listdir(CSRC) if n.endswith((".hip", ".cpp")) and n != "ops_binding.cpp"]
    headers = {h for n in sources for h in included(n)}
    assert {"philox.h", "short_tiles.h", "../../include/gpt_hip.h"} <= headers
    for header in headers:
        built = would_build("-W", header)
        for n in sources:
            if header in included(n):
                assert re.search(rf" -c {re.escape(n)} ", built), (header, n)


def test_another_torch_rebuilds_the_binding(tmp_path):
    """The binding is compiled against torch's headers: one built for the torch that is there is kept, another torch makes a new one.  The
    compiler is a script that notes its runs, the torch a folder with a version."""
    compiler, runs, binding = tmp_path / "cxx", tmp_path / "runs", str(tmp_path / "gpt_ops.so")
    compiler.write_text(f'#!/bin/sh\necho run >> {runs}\nwhile [ "$1" != -o ]; do shift; done\necho built > "$2"\n')
    compiler.chmod(0o755)
    (tmp_path / "torch").mkdir()
    (tmp_path / "torch" / "__init__.py").write_text("")

    def make(version):
        (tmp_path / "torch" / "version.py").write_text(f"__version__ = {version!r}\n")
        subprocess.run(["make", "-C", CSRC, binding, "BIND=" + binding, f"CXX={compiler}", f"PYTHON=env PYTHONPATH={tmp_path} python3"], check=True,
                       capture_output=True)
        return len(runs.read_text().split())
    assert [make(v) for v in ("1", "1", "2", "2", "1")] == [1, 1, 2, 2, 3]


def test_the_c_library_needs_no_torch():
    without = "PYTHON=python3 -I -S"                                     # no site-packages, so no torch
    for args in (["lib"], ["all", without], [without]):
        listed = would_build(*args, "-B")
        assert "-o ../lib/libgpt_hip.so" in listed and "ops_binding.cpp" not in listed, args
    assert "ops_binding.cpp" in would_build("-B")
