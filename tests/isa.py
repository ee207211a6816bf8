"""The device code of the built library, disassembled: instructions with their
predecessors, so that what the hardware leaves to software can be checked on
code that inline assembly took out of the compiler's hands."""
import os
import re
import struct
import subprocess
import tempfile
from collections import defaultdict
from typing import NamedTuple

ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
OBJDUMP = os.path.join(ROCM, "llvm", "bin", "llvm-objdump")
_MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


class Instruction(NamedTuple):
    kernel: str
    op: str
    args: str


def code_objects(path: str, arch: str = "gfx950"):
    """The code objects for `arch` in a library's offload bundles."""
    data = open(path, "rb").read()
    at = data.find(_MAGIC)
    while at >= 0:
        (count,) = struct.unpack_from("<Q", data, at + 24)
        p = at + 32
        for _ in range(count):
            offset, size, name = struct.unpack_from("<QQQ", data, p)
            target = data[p + 24:p + 24 + name].decode()
            p += 24 + name
            if target.endswith(arch) and size:
                yield data[at + offset:at + offset + size]
        at = data.find(_MAGIC, at + 8)


def disassembled(code: bytes):
    """(instructions, predecessors by index) of one code object."""
    with tempfile.NamedTemporaryFile(suffix=".co") as f:
        f.write(code)
        f.flush()
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", f.name], check=True, stdout=subprocess.PIPE, text=True).stdout
    ins, place, targets = [], {}, []
    before = defaultdict(list)
    kernel, start, falls = "", 0, False
    for line in text.splitlines():
        head = re.match(r"^([0-9a-f]{16}) <(.*)>:", line)
        if head:
            kernel, start, falls = head.group(2), int(head.group(1), 16), False
            continue
        m = re.match(r"^\t(\S+)\s*(.*?)\s*// ([0-9A-F]+): [0-9A-F ]+(<\S+?(?:\+0x([0-9a-f]+))?>)?", line)
        if not m:
            continue
        op, i = m.group(1), len(ins)
        ins.append(Instruction(kernel, op, m.group(2)))
        place[int(m.group(3), 16)] = i
        if falls:
            before[i].append(i - 1)
        falls = op not in ("s_branch", "s_endpgm", "s_setpc_b64")
        if op.startswith(("s_branch", "s_cbranch")):
            assert m.group(4), line
            targets.append((i, start + int(m.group(5) or "0", 16)))
    for i, t in targets:
        before[place[t]].append(i)
    return ins, before


def scalars(arg: str) -> set:
    """The scalar registers that an operand names."""
    found = set()
    for lo, hi in re.findall(r"\bs\[(\d+):(\d+)\]", arg):
        found.update(f"s{i}" for i in range(int(lo), int(hi) + 1))
    found.update(re.findall(r"\bs\d+\b", arg))
    if re.search(r"\bvcc\b", arg):
        found.update(("vcc_lo", "vcc_hi"))
    found.update(re.findall(r"\b(?:vcc_lo|vcc_hi|m0)\b", arg))
    return found


def writers(ins, before, i: int, states: int):
    """The instructions fewer than `states` wait states before instruction i,
    on any path."""
    best, stack = {}, [(p, 0) for p in before[i]]
    while stack:
        j, waited = stack.pop()
        if waited >= states or best.get(j, states) <= waited:
            continue
        best[j] = waited
        yield ins[j]
        step = int(ins[j].args, 0) + 1 if ins[j].op == "s_nop" else 1
        stack.extend((p, waited + step) for p in before[j])
