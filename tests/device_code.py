"""The gfx950 code of a library built here, as its compiler's own tools list
it: instructions with the addresses that branches name, and the kernels'
resources."""
import collections
import glob
import os
import re
import shutil
import subprocess

LLVM = os.environ.get("Q38M_LLVM_BIN", "/opt/rocm/llvm/bin")

Instruction = collections.namedtuple("Instruction", "address name operands kernel")


def code_objects(library, directory):
    """The device code objects of a library, extracted into an empty directory."""
    copy = os.path.join(str(directory), "lib.so")
    shutil.copy(library, copy)
    subprocess.run([os.path.join(LLVM, "llvm-objdump"), "--offloading", copy], check=True,
                   capture_output=True)
    return sorted(p for p in glob.glob(copy + ".*gfx950*") if os.path.getsize(p))


def resources(code_object):
    """Kernel name -> its metadata's whole numbers."""
    notes = subprocess.run([os.path.join(LLVM, "llvm-readelf"), "--notes", code_object], check=True,
                           capture_output=True, text=True).stdout
    found = {}
    for entry in re.split(r"\n  - ", notes)[1:]:
        name = re.search(r"\.name: +(_Z\S+)", entry)
        if name:
            found[name.group(1)] = {k: int(v) for k, v in re.findall(r"\.(\w+): +(\d+)\s*$", entry, re.M)}
    return found


def parse(text):
    """Instructions of a listing, in order of their addresses."""
    kernel, out = None, []
    for line in text.splitlines():
        head = re.match(r"[0-9a-fA-F]+ <(\S+)>:", line)
        if head:
            kernel = head.group(1)
            continue
        body = re.match(r"\s+(\S+)(?:\s+(.*?))?\s*// ([0-9A-Fa-f]+):", line)
        if body:
            operands = tuple(o.strip() for o in (body.group(2) or "").split(","))
            out.append(Instruction(int(body.group(3), 16), body.group(1), operands, kernel))
    return out


def disassemble(code_object):
    return parse(subprocess.run([os.path.join(LLVM, "llvm-objdump"), "-d", "--mcpu=gfx950", code_object],
                                check=True, capture_output=True, text=True).stdout)


def scalar_registers(operand):
    """Names of the scalar registers that an operand's text holds."""
    found = set()
    for low, high in re.findall(r"(?<![a-z])s\[(\d+):(\d+)\]", operand):
        found.update(f"s{i}" for i in range(int(low), int(high) + 1))
    found.update(re.findall(r"(?<![a-z0-9_])s\d+", operand))
    for name in ("vcc", "m0"):
        if re.search(rf"(?<![a-z0-9_]){name}(?![a-z0-9])", operand):
            found.add(name)
    return found


def vector_writes(i):
    """Scalar registers that a vector instruction writes: its first operand, and the second of
    those with a carry or a scale flag."""
    if not i.name.startswith("v_"):
        return set()
    count = 2 if re.search(r"_co_|v_mad_[iu]64|v_div_scale", i.name) else 1
    return set().union(*(scalar_registers(o) for o in i.operands[:count]))


def memory_reads(i):
    """Scalar registers that a vector memory instruction reads."""
    if not re.match(r"(global|buffer|scratch|flat)_", i.name):
        return set()
    return set().union(*(scalar_registers(o) for o in i.operands))


def too_soon(instructions, reads, writes, wait_states):
    """[(writer, reader)]: readers with fewer than `wait_states` wait states between a write of a
    register and their read of it, on any way through the branches.  An instruction is a wait
    state, s_nop n is n + 1."""
    at = {i.address: k for k, i in enumerate(instructions)}
    before = collections.defaultdict(list)
    for k, i in enumerate(instructions):
        if re.match(r"s_(c?branch|call)", i.name) and re.fullmatch(r"\d+", i.operands[-1]):
            jump = int(i.operands[-1])
            to = at.get(i.address + 4 + 4 * (jump - 65536 if jump >= 32768 else jump))
            if to is not None:
                before[to].append(k)
        if k + 1 < len(instructions) and i.name not in ("s_branch", "s_endpgm", "s_setpc_b64"):
            before[k + 1].append(k)
    found = []
    for k, i in enumerate(instructions):
        wanted = reads(i)
        if not wanted:
            continue
        open_ways, seen = [(p, 0) for p in before[k]], set()
        while open_ways:
            p, passed = open_ways.pop()
            if passed >= wait_states or (p, passed) in seen:
                continue
            seen.add((p, passed))
            writer = instructions[p]
            if writes(writer) & wanted:
                found.append((writer, i))
            states = int(writer.operands[0]) + 1 if writer.name == "s_nop" else 1
            open_ways += [(q, passed + states) for q in before[p]]
    return found
