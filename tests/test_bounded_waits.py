"""How the warp-specialised kernels leave their waits, read from their source:
a wait that ran out marks its CTA dead, and every role has to come to the
block's last barrier all the same.  Nothing here runs on a GPU: a kernel whose
wait runs out is not made to."""

from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "ervf_b200" / "csrc"
KERNELS = ["linear.cu", "ssm_chunk.cu"]


def stripped(name):
    """The source without comments and strings, line by line."""
    s = (CSRC / name).read_text()
    s = re.sub(r'"(\\.|[^"\\\n])*"', '""', s)
    s = re.sub(r"/\*.*?\*/", lambda m: "\n" * m.group().count("\n"), s, flags=re.S)
    return [re.sub(r"//.*", "", line) for line in s.split("\n")]


def blocks_around(lines):
    """For each line the heads of the brace blocks that it stands in."""
    stack, around, head = [], [], ""
    for line in lines:
        around.append([*stack, line])
        for ch in line:
            if ch == "{":
                stack.append(head)
                head = ""
            elif ch == "}":
                stack and stack.pop()
                head = ""
            elif ch == ";" and head.count("(") == head.count(")"):  # not a loop's own
                head = ""
            else:
                head += ch
    return around


@pytest.mark.parametrize("name", KERNELS)
def test_dead_is_read_by_single_lanes_and_by_the_waits_alone(name):
    """The flag may change between two lanes' reads, so no branch or loop of a whole warp goes by it:
    lanes that left would meet the others at no warp-wide instruction any more."""
    lines = stripped(name)
    reads = 0
    for at, around in zip(lines, blocks_around(lines)):
        if re.search(r"(if|for|while)\s*\(.*\*dead\b(?!\s*=[^=])", at):
            reads += 1
            alone = any(re.search(r"lane == 0|tid == 0|lin_wait_slow", h) for h in around)
            assert alone, f"{name}: a whole warp branches on the flag: {at.strip()}"
    assert reads


def test_no_tensor_copy_outlives_a_dead_cta():
    """The loop behind a producer's last load waits for the copies in flight: by their arrival, or,
    where it goes by waits that a dead CTA ends at once, by the clock behind it."""
    lines = stripped("linear.cu")
    drains = [i for i, line in enumerate(lines) if "k = loads >" in line]
    assert len(drains) == 2
    for i in drains:
        by_arrival = re.search(r"\bmbar_wait\(", lines[i + 1])
        by_clock = "*dead" in lines[i + 2] and "clock64()" in "".join(lines[i + 3:i + 5])
        assert by_arrival or by_clock, lines[i + 1].strip()
