"""Static guard for the matrix instructions that csrc/mx_gemm.hip's large tile issues through inline asm (CPU only:
disassembles the library built here).

The compiler does not know what an asm statement is, so it leaves out the wait states that the hardware needs around a
matrix instruction: behind it, before anything but the next link of the same sum touches its result; in front of it,
behind a vector instruction that writes one of its operands.  The kernel's own waits cover the places where that happens,
and this check fails if the compiler's order of instructions ever makes another one.  Both sides of every branch are
followed."""
import os
import re

import pytest
from test_isa_hazards import _device_disassembly, _regs

BEHIND = 20     # wait states: a matrix instruction of 16 passes, and four to read its result
BEFORE = 2      # a vector instruction's result as a matrix operand
KERNEL = "mx_gemm_large_kernel"


def parse(text):
    """{function: [(address, opcode, operands, branch target or None, text)]} of the large tile's kernels."""
    funcs, insts, base = {}, None, 0
    for line in text.splitlines():
        m = re.match(r"^([0-9a-f]+) <([^>]+)>:", line)
        if m:
            base = int(m.group(1), 16)
            insts = funcs.setdefault(m.group(2), []) if KERNEL in m.group(2) else None
            continue
        if insts is None or "//" not in line:
            continue
        body, note = line.split("//", 1)
        parts = body.strip().split(None, 1)
        if not parts:
            continue
        ops = [o.strip() for o in parts[1].split(",")] if len(parts) > 1 else []
        address = int(note.split(":")[0], 16)
        target = re.search(r"<[^>+]+(?:\+0x([0-9a-f]+))?>", note) if "branch" in parts[0] else None
        insts.append((address, parts[0], ops, base + int(target.group(1) or "0", 16) if target else None, body.strip()))
    return funcs


def touched(ops):
    return set().union(*[_regs(o.split()[0]) for o in ops if o]) if ops else set()


def cost(op, ops):
    return 1 + (int(ops[0]) if op == "s_nop" else 0)


def walk(insts, at, need, visit):
    """Calls visit(inst) on what can run within `need` wait states behind instruction `at`; True from it ends a path."""
    index = {inst[0]: i for i, inst in enumerate(insts)}
    todo, seen = [(at + 1, 0)], {}
    while todo:
        i, states = todo.pop()
        while i < len(insts) and states < need and seen.get(i, need) > states:
            seen[i] = states
            _, op, ops, target, _ = insts[i]
            if visit(insts[i]) or op == "s_endpgm":
                break
            states += cost(op, ops)
            if target is not None:
                todo.append((index[target], states))
                if op == "s_branch":
                    break
            i += 1


def violations(text):
    bad, links = [], 0
    for name, insts in parse(text).items():
        for at, inst in enumerate(insts):
            _, op, ops, _, body = inst
            if op.startswith("v_mfma"):
                links += 1
                dst = _regs(ops[0])

                def visit(other):
                    _, op2, ops2, _, body2 = other
                    if op2.startswith("v_mfma") and _regs(ops2[0]) == dst and not touched(ops2[1:3] + ops2[4:]) & dst:
                        return True
                    if touched(ops2) & dst:
                        bad.append((name, body, body2))
                        return True
                    return False

                walk(insts, at, BEHIND, visit)
            elif op.startswith("v_") and not op.startswith("v_cmp") and ops:
                dst = _regs(ops[0].split()[0])

                def visit(other):
                    _, op2, ops2, _, body2 = other
                    if op2.startswith("v_mfma") and touched(ops2) & dst:
                        bad.append((name, body, body2))
                        return True
                    return False

                walk(insts, at, BEFORE, visit)
    return bad, links


SAMPLE = """
0000000000001000 <x_mx_gemm_large_kernel_y>:
	v_mov_b32_e32 v30, v31   // 000000001000: 00000000
	{first}   // 000000001004: 00000000
	v_mfma_f32_16x16x32_bf16 v[10:13], v[20:23], v[30:33], v[10:13]   // 000000001008: 00000000
	v_mfma_f32_16x16x32_bf16 v[10:13], v[20:23], v[34:37], v[10:13]   // 000000001010: 00000000
	s_cbranch_scc1 65530   // 000000001018: BF850000 <x_mx_gemm_large_kernel_y+{target}>
	s_nop 15   // 00000000101C: 00000000
	s_nop 15   // 000000001020: 00000000
	v_max_f32_e32 v40, 0, v11   // 000000001024: 00000000
	s_endpgm   // 000000001028: 00000000
	ds_read_b128 v[12:15], v1   // 00000000102C: 00000000
	s_endpgm   // 000000001030: 00000000
"""


@pytest.mark.parametrize("first, target, count", [("s_nop 1", "0x8", 0), ("s_nop 0", "0x8", 1), ("s_nop 1", "0x2c", 1),
                                                  ("s_nop 1", "0x24", 1)])
def test_checker(first, target, count):
    assert len(violations(SAMPLE.format(first=first, target=target))[0]) == count


def test_large_tile_waits_for_its_matrix_instructions():
    found = [violations(text) for text in _device_disassembly()]
    bad = [b for f in found for b in f[0]]
    assert not bad, "\n".join("%s: '%s' then '%s'" % b for b in bad[:20])
    assert sum(f[1] for f in found) >= 64
