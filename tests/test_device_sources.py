"""What the device sources may hold.  Global memory is written through vector stores only -- plain C++ stores, which the compiler turns
into them; the scalar unit's data cache is a read path.  The compiler never writes through it by itself, so the one way in is inline
assembly: every instruction in it is a VALU instruction or one of the few scalar ones that touch registers alone."""
import glob
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCES = sorted(os.path.relpath(path, ROOT) for pattern in ("shasta_amd/csrc/*.h*", "scripts/**/*.h*", "include/*.h") for path in glob.glob(os.path.join(ROOT, pattern), recursive=True))

STATEMENT = re.compile(r"\b(?:asm|__asm__|__asm)\b\s*(?:volatile|__volatile__|goto|inline)?\s*\(\s*((?:\"(?:[^\"\\]|\\.)*\"\s*)+)")
STRING = re.compile(r"\"((?:[^\"\\]|\\.)*)\"")
REGISTERS_ONLY = {"s_mov_b32", "s_nop", "s_waitcnt", "llvm.amdgcn.writelane.i32"}        # (the last: the label of a declaration that names a compiler intrinsic)


def without_comments(text):
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


def assembly_mnemonics(text):
    mnemonics = []
    for statement in STATEMENT.finditer(without_comments(text)):
        lines = "".join(s.group(1) for s in STRING.finditer(statement.group(1))).replace("\\n", "\n").replace("\\t", " ")
        mnemonics += [line.split()[0] for line in re.split(r"[\n;]", lines) if line.split()]
    return mnemonics


def test_the_reading_of_inline_assembly():
    text = 'asm volatile("v_add_u32 %0, %0, %1\\n\\ts_nop 0" : "+v"(a)); // asm("v_commented_out")\n  asm("v_mov_b32 %0, 1\\n" "v_xor_b32 %0, %0, 2" : "=v"(b));'
    assert assembly_mnemonics(text) == ["v_add_u32", "s_nop", "v_mov_b32", "v_xor_b32"]


def test_the_device_sources_are_found():
    assert "shasta_amd/csrc/primitives.hpp" in SOURCES and "shasta_amd/csrc/align4.hip" in SOURCES and "scripts/microbench/valu_rates.hip" in SOURCES


@pytest.mark.parametrize("path", SOURCES)
def test_inline_assembly_writes_no_memory(path):
    text = open(os.path.join(ROOT, path)).read()
    mnemonics = assembly_mnemonics(text)
    assert len(STATEMENT.findall(without_comments(text))) == len(re.findall(r"\b(?:asm|__asm__|__asm)\b", without_comments(text)))      # (none is left unread)
    assert [m for m in mnemonics if not (m.startswith("v_") or m in REGISTERS_ONLY)] == []


def test_every_device_source_is_compiled_without_packed_fp32_instructions():
    lines = subprocess.run(["make", "-n", "-B", "-C", os.path.join(ROOT, "shasta_amd", "csrc")], capture_output=True, text=True, check=True).stdout.splitlines()
    compiled = [line for line in lines if "hipcc" in line and " -c " in line]
    assert sorted(re.search(r"-c (\S+\.hip)", line).group(1) for line in compiled) == sorted(os.path.basename(path) for path in SOURCES if path.startswith("shasta_amd/csrc") and path.endswith(".hip"))
    assert all("-Xclang -target-feature -Xclang -packed-fp32-ops" in line for line in compiled)
