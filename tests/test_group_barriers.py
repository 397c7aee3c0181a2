"""Barriers of some of a block's warps, read from the sources (no GPU).

A bounded wait runs out for each warp by itself.  A warp that leaves its loop at once then leaves the others at the next barrier of their group, for
good: where a loop holds such a barrier, the warps decide together (a vote on the outcome of the wait), or the loop needs no barrier."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "llama3-custom-inference_b200" / "csrc"
BARRIER = re.compile(r'"[^"\n]*\bbar\.(?:sync|red)\b|(?<!auto )(?<!void )\b(?:meet|sync_compute|output_warps_meet|output_warps_agree)\(')
LEAVES = re.compile(r"\{ ok = false; break; \}")


def code_of(text):
    """Comments blanked, places kept."""
    return re.sub(r"//[^\n]*", lambda m: " " * len(m.group()), text)


def loops_around(code, at):
    """The bodies (begin, end) of the loops that hold place `at`."""
    opened, pairs = [], []
    for i, c in enumerate(code):
        if c == "{":
            opened.append(i)
        elif c == "}" and opened:
            pairs.append((opened.pop(), i))
    for begin, end in pairs:
        if begin < at < end:
            head = code[max(code.rfind(";\n", 0, begin), code.rfind("}\n", 0, begin), code.rfind("{\n", 0, begin), 0):begin]
            if re.search(r"\b(for|while)\s*\(", head):
                yield begin, end


def left_alone(text):
    code = code_of(text)
    return sorted({code.count("\n", 0, m.start()) + 1 for m in BARRIER.finditer(code) for begin, end in loops_around(code, m.start()) if LEAVES.search(code, begin, end)})


def test_the_check_itself():
    loop = 'void k() {\n  for (;;) {\n    if (!wait()) { ok = false; break; }\n    for (int e = 0; e < 2; ++e) {\n      asm volatile("bar.sync 2, 128;");\n    }\n  }\n}\n'
    assert left_alone(loop) == [5]
    assert left_alone(loop.replace("{ ok = false; break; }", "ok = false;")) == []
    assert left_alone(loop.replace("  for (;;) {\n", "  for (;;) {\n  }\n  {\n")) == []


@pytest.mark.parametrize("name", sorted(p.name for p in CSRC.glob("*.cu")))
def test_no_warp_leaves_the_others_at_a_barrier(name):
    assert left_alone((CSRC / name).read_text()) == []
