"""Wait states that the gfx950 instruction set asks of the program, in the instructions of the built library.
The compiler sees to them in its own code and does not look into asm strings."""
from __future__ import annotations

import os
import re
import struct
import subprocess

import pytest

from conftest import PKG_DIR

LIB = os.path.join(PKG_DIR, "libdgm_amd.so")
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def code_objects():
    """The device code in the library: bundles of (offset, size, target)."""
    data = open(LIB, "rb").read()
    at = data.find(MAGIC)
    while at >= 0:
        count, = struct.unpack_from("<Q", data, at + 24)
        p = at + 32
        for _ in range(count):
            offset, size, n = struct.unpack_from("<QQQ", data, p)
            if data[p + 24:p + 24 + n].endswith(b"gfx950") and size:
                yield data[at + offset:at + offset + size]
            p += 24 + n
        at = data.find(MAGIC, at + 24)


def scalars(operand):
    """The numbers of the scalar registers that an operand names."""
    m = re.match(r"s(?:\[(\d+):(\d+)\]|(\d+)\b)", operand.strip())
    if not m:
        return set()
    return {int(m[3])} if m[3] else set(range(int(m[1]), int(m[2]) + 1))


def states(op, args):
    return int(args, 0) + 1 if op == "s_nop" else 1


def faults(listing):
    """(copies into LDS, what is too close) of one disassembly."""
    copies, found, kernel, past = 0, [], "", []
    for line in listing.splitlines():
        m = re.match(r"[0-9a-f]+ <(.*)>:", line)
        if m:
            kernel, past = m[1], []
            continue
        m = re.match(r"\s+([a-z]\w+) ?(.*?)\s*(?://.*)?$", line)
        if not m:
            continue
        op, args = m[1], m[2]
        if op.startswith(("global_", "buffer_")):
            copy = "_lds_" in op or args.endswith(" lds")
            copies += copy
            read, waited = set(), 0
            for operand in args.split(","):
                read |= scalars(operand)
            for o, a in reversed(past):
                to = a.split(",")[0]
                if copy and waited < 1 and to.strip() == "m0":
                    found.append((kernel, "m0", o, a, op, args))
                if o.startswith("v_") and scalars(to) & read:
                    found.append((kernel, "scalar written by a vector instruction", o, a, op, args))
                waited += states(o, a)
                if waited >= 5:
                    break
        past = past[-7:] + [(op, args)]
    return copies, found


PATTERN = """
0000000000001000 <kernel>:
\ts_mov_b32 m0, s4      // 000000001000: BEFC0004
{between}\tglobal_load_lds_dwordx4 v1, s[8:9] // 000000001004: DDF48000 00080001
"""


@pytest.mark.parametrize("between,bad", [
    ("", 1), ("\ts_nop 0   // 1: 0\n", 0), ("\tv_mov_b32_e32 v3, v4\n", 0), ("\ts_nop 0\n\ts_nop 0\n", 0),
    ("\tv_readfirstlane_b32 s8, v0\n\ts_nop 3\n", 1), ("\tv_readlane_b32 s9, v0, 3\n\ts_nop 4\n", 0),
    ("\tv_readfirstlane_b32 s10, v0\n", 0)])
def test_the_reader_finds_what_is_too_close(between, bad):
    copies, found = faults(PATTERN.format(between=between))
    assert copies == 1 and len(found) == bad


def test_copies_into_lds_wait_for_what_they_read():
    """One wait state from a scalar write of m0 to a copy into LDS; five from a vector instruction's write of a scalar
    register to the memory instruction that takes it."""
    copies, found = 0, []
    for obj in code_objects():
        done = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "-"], input=obj, capture_output=True)
        assert done.returncode == 0, done.stderr
        n, f = faults(done.stdout.decode())
        copies += n
        found += f
    assert copies > 0, "the library's copies into LDS were not found"
    assert not found, f"{len(found)} of {copies} copies, the first: {found[0]}"
