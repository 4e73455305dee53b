"""The machine code of the operators' library, as it was built here from source: what its hand-written memory instructions need around them, which the
compiler does not see."""
import os
import re
import shutil
import subprocess

import pytest

from hsenet_amd import _ops as O
from hsenet_amd.build import build

OBJDUMP = shutil.which("llvm-objdump") or "/opt/rocm/llvm/bin/llvm-objdump"
pytestmark = pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no llvm-objdump")


@pytest.fixture(scope="module")
def listings(tmp_path_factory):
    """the gfx950 code of each source file, disassembled"""
    build()
    O.check_fresh()
    at = tmp_path_factory.mktemp("code")
    shutil.copy(O.LIB_PATH, at / "ops.so")
    subprocess.run([OBJDUMP, "--offloading", "ops.so"], cwd=at, check=True, capture_output=True)
    objects = [f for f in os.listdir(at) if f.endswith("gfx950")]
    assert len(objects) == 3
    return [subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", f], cwd=at, check=True, capture_output=True, text=True).stdout for f in objects]


def parsed(listing):
    """[(operation, operands)] and, for each of them, the numbers of those that may run right before it; a symbol is an operation \"\" """
    ops, where, jumps = [], {}, []
    for line in listing.splitlines():
        m = re.match(r"\t(\S+)(.*?)\s+// ([0-9A-F]+):", line)
        if m:
            to = re.search(r"<(\S+?)(?:\+0x([0-9a-f]+))?>$", line)
            if to and "branch" in m[1]:
                jumps.append((len(ops), to[1], int(to[2] or "0", 16)))
            where[int(m[3], 16)] = len(ops)
            ops.append((m[1], m[2]))
        elif m := re.match(r"([0-9a-f]+) <(\S+)>:", line):
            where[m[2]] = int(m[1], 16)
            ops.append(("", m[2]))
    before = [[i - 1] if i and ops[i - 1][0] not in ("s_branch", "s_endpgm", "s_setpc_b64") and ops[i][0] else [] for i in range(len(ops))]
    for i, symbol, offset in jumps:
        before[where[where[symbol] + offset]].append(i)
    return ops, before


def scalars(operands):
    out = set()
    for first, last, one in re.findall(r"\bs\[(\d+):(\d+)\]|\bs(\d+)\b", operands):
        out |= {int(one)} if one else set(range(int(first), int(last) + 1))
    return out


def too_near(listing, need):
    """(memory instruction, the vector instruction that writes a scalar register of its) with fewer than `need` wait states between them, on any path"""
    ops, before = parsed(listing)
    found, seen = [], 0
    for i, (op, operands) in enumerate(ops):
        if not re.match(r"(buffer|global|flat|scratch)_", op):
            continue
        seen += 1
        read, todo = scalars(operands), [(j, 0) for j in before[i]]
        while read and todo:
            j, waited = todo.pop()
            if waited >= need:
                continue
            name, x = ops[j]
            if name.startswith("v_") and read & scalars(x.split(",")[0]):
                found.append((op + operands, name + x))
                break
            todo += [(k, waited + (int(x) + 1 if name == "s_nop" else 1 if name else 0)) for k in before[j]]
    return found, seen


def test_scalar_operands_of_memory_instructions_have_settled(listings):
    """a memory instruction may read a scalar register that a vector instruction wrote (v_readfirstlane) five wait states later at the earliest"""
    total = 0
    for text in listings:
        found, seen = too_near(text, 5)
        total += seen
        assert not found, f"{len(found)} in all, the first: {found[0]}"
    assert total > 1000
    # the check sees what it is for
    head = "0000000000000100 <f>:\n\tv_readfirstlane_b32 s29, v6    // 000000000100: 0\n"
    tail = "\tbuffer_load_dwordx4 v7, s[12:15], s29 offen lds    // 000000000110: 0\n"
    assert len(too_near(head + "\ts_mov_b32 m0, s28    // 000000000104: 0\n\ts_nop 0    // 000000000108: 0\n" + tail, 5)[0]) == 1
    assert not too_near(head + "\ts_mov_b32 m0, s28    // 000000000104: 0\n\ts_nop 3    // 000000000108: 0\n" + tail, 5)[0]


def test_transfers_to_lds_set_m0_in_time(listings):
    """M0 holds the place in LDS: one wait state at least between its write and the transfer, on any path"""
    count = 0
    for text in listings:
        ops, before = parsed(text)
        for i, (op, operands) in enumerate(ops):
            if op.startswith("buffer_load") and operands.rstrip().endswith("lds"):
                count += 1
                assert all(not (ops[j][1].split(",")[0].strip() == "m0") for j in before[i]), ops[i]
    assert count > 100
