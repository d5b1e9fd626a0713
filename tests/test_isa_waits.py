"""The built library's machine code keeps the distances that the hardware does
not: a vector memory instruction reads a scalar register that a vector
instruction wrote no sooner than 5 wait states later, and m0 no sooner than 1
after it was set where it loads to LDS. The compiler sees to both in code of its
own, but not across the edge of a statement of inline assembly."""
import os
import re
import shutil
import struct
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "eccv26_tad_amd", "libsvtad_sparse.so")
LLVM = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin")
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"
NEEDED = 5


def _code_objects(path):
    """The gfx950 code objects of a host library's offload bundles."""
    data = open(path, "rb").read()
    at = data.find(MAGIC)
    while at >= 0:
        (entries,) = struct.unpack_from("<Q", data, at + len(MAGIC))
        pos = at + len(MAGIC) + 8
        if entries > 64:  # the magic as a string, no bundle
            entries = 0
        for _ in range(entries):
            offset, size, n = struct.unpack_from("<QQQ", data, pos)
            name = data[pos + 24 : pos + 24 + n]
            pos += 24 + n
            if b"gfx950" in name and size:
                yield data[at + offset : at + offset + size]
        at = data.find(MAGIC, at + 1)


def _scalars(operand):
    """The scalar registers that an operand names."""
    m = re.fullmatch(r"s\[(\d+):(\d+)\]", operand)
    if m:
        return set(range(int(m[1]), int(m[2]) + 1))
    m = re.fullmatch(r"s(\d+)", operand)
    return {int(m[1])} if m else {"vcc"} if operand == "vcc" else {"m0"} if operand == "m0" else set()


def hazards(listing):
    """The vector memory instructions of a disassembly that come too soon after
    what they read, as (line, wait states), and how many there were to look at."""
    found, seen = [], 0
    vector, m0 = {}, 99  # wait states since a vector instruction wrote a scalar register, since m0 was set
    for line in listing:
        op, _, rest = line.split("//")[0].strip().partition(" ")
        if not op or op.endswith(":") or not re.match(r"(s|v|ds|buffer|global|flat|scratch)_", op):
            if op.endswith(":"):
                vector, m0 = {}, 99
            continue
        operands = [o.strip().split(" ")[0] for o in rest.split(",")]
        if op.startswith(("buffer_", "global_", "flat_", "scratch_")):
            seen += 1
            for o in operands:
                for s in _scalars(o):
                    if vector.get(s, 99) < NEEDED:
                        found.append((line.strip(), vector[s]))
            if rest.split("//")[0].strip().endswith(" lds") and m0 < 1:
                found.append((line.strip(), m0))
        states = int(rest.strip(), 0) + 1 if op == "s_nop" else 1
        vector = {k: n + states for k, n in vector.items() if n + states < NEEDED}
        m0 += states
        if op.startswith("v_") and operands:
            written = operands[:2] if re.search(r"_(co|co_ci)_", op) or op.startswith("v_div_scale") else operands[:1]
            for o in written:
                for s in _scalars(o):
                    vector[s] = 0
        elif op.startswith("s_") and operands:
            for s in _scalars(operands[0]):
                vector.pop(s, None)
                if s == "m0":
                    m0 = 0
    return found, seen


def test_the_check_itself():
    def run(*lines):
        return [n for _, n in hazards(lines)[0]]

    load = "\tbuffer_load_dword v50, s[36:39], 0 offen lds  // 0000: E0511000"
    write = "\tv_readfirstlane_b32 s36, v92"
    assert run(write, "\ts_and_b32 s37, s37, 0xffff", "\ts_mov_b32 m0, s79", "\ts_nop 0", load) == [3]
    assert run(write, "\ts_and_b32 s37, s37, 0xffff", "\ts_mov_b32 m0, s79", "\ts_nop 2", load) == []
    assert run(write, "\ts_mov_b32 s36, 0", load) == []
    assert run("\tv_cmp_gt_i32_e64 s[38:39], v1, v2", load) == [0, 0]
    assert run("\ts_mov_b32 m0, s79", load) == [0]
    assert run("\tv_mov_b32_e32 v50, v1", load) == []


def test_library():
    objdump = os.path.join(LLVM, "llvm-objdump")
    if not os.path.exists(objdump):
        objdump = shutil.which("llvm-objdump")
    if not objdump:
        pytest.skip("no llvm-objdump")
    if not os.path.exists(LIB):
        pytest.fail("libsvtad_sparse.so not built (run python eccv26_tad_amd/build.py)")
    seen = 0
    for code in _code_objects(LIB):
        r = subprocess.run([objdump, "-d", "-"], input=code, stdout=subprocess.PIPE, check=True)
        found, n = hazards(r.stdout.decode().splitlines())
        seen += n
        assert not found, found[:5]
    assert seen > 1000
