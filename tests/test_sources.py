"""Rules of the kernels' sources that the compiler does not check."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "burnisher_amd" / "csrc"
MEMORY = re.compile(r"(global|flat|buffer|scratch|tbuffer)_")


def assembly(text):
    """(instructions, constraint of each operand) of every asm statement."""
    for body in re.findall(r'\basm\s*(?:volatile\s*)?\((.*?)\)\s*;', text, re.S):
        template = "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', body.split(":")[0]))
        constraints = re.findall(r'"([=+&]*[a-z0-9]+)"\s*\(', body)
        yield [i.strip() for i in re.split(r"\\n|\\t|;", template) if i.strip()], constraints


def waits_for_scalar_addresses(text):
    """Per memory instruction of inline assembly that reads a scalar operand: the wait states before it in its own block,
    None where the block's own scalar move wrote the operand."""
    found = []
    for instructions, constraints in assembly(text):
        states, moved = 0, set()
        for i in instructions:
            operands = [int(x) for x in re.findall(r"%(\d+)", i)]
            scalar = [o for o in operands if "s" in constraints[o]]
            if MEMORY.match(i) and scalar:
                found.append(None if set(scalar) <= moved else states)
            if i.startswith("s_mov_b64"):
                moved.add(operands[0])
            nop = re.match(r"s_nop (\d+)", i)
            states += int(nop.group(1)) + 1 if nop else 1
    return found


def test_the_rule_sees_what_it_looks_for():
    form = 'asm volatile("s_mov_b32 m0, %0\\n\\ts_nop {}\\n\\tglobal_load_lds_dwordx4 %1, {}" : : "s"(l), "v"(o), "s"(b) : "memory");'
    assert waits_for_scalar_addresses(form.format(0, "%2")) == [2]
    assert waits_for_scalar_addresses(form.format(4, "%2")) == [6]
    assert waits_for_scalar_addresses(form.format(0, "off")) == []
    form = 'asm volatile("s_mov_b64 %0, %{}\\n\\tglobal_load_dword %1, %{}" : "=&s"(t) : "v"(o), "s"(b));'
    assert waits_for_scalar_addresses(form.format(2, 0)) == [None]
    assert waits_for_scalar_addresses(form.format(2, 2)) == [1]


@pytest.mark.parametrize("path", sorted(p.name for p in CSRC.iterdir()))
def test_memory_instructions_wait_for_a_scalar_address(path):
    # A vector instruction that wrote a scalar register (a readlane of a spilled address) is five wait states ahead
    # of a memory instruction that reads it, and the compiler adds none inside or before inline assembly. Scalar
    # instructions are ordered by the hardware.
    assert all(n is None or n >= 5 for n in waits_for_scalar_addresses((CSRC / path).read_text()))


@pytest.mark.parametrize("path", sorted(p.name for p in CSRC.iterdir()))
def test_workgroup_numbers_are_compared_before_they_are_narrowed(path):
    # the last row of a launch along y may count past 2^31
    assert not re.search(r"(static_cast<(unsigned|int|u?int32_t)>|\(int\)|\bint \w+ = |\bunsigned \w+ = )\s*\(?group_index\(\)",
                         (CSRC / path).read_text())


def test_direct_loads_with_a_scalar_address_are_found():
    assert len(waits_for_scalar_addresses((CSRC / "common.h").read_text())) == 2
