"""CPU test of the inline-assembly copies into LDS: each begins with the wait states that its scalar operands need.

A buffer instruction must not read a scalar register within five wait states of a vector instruction's write of it; the
compiler keeps that for its own instructions only, and may bring a spilled operand back with v_readlane right before the
assembly. ``s_nop 4`` is five wait states.
"""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "memopt-transformer-runtime_amd", "csrc")


def statements():
    """(file, text) of every inline-assembly statement that copies into LDS (they take m0)."""
    for name in sorted(os.listdir(CSRC)):
        text = open(os.path.join(CSRC, name)).read()
        text = re.sub(r"//[^\n]*", "", text)
        for m in re.finditer(r"\basm\s+volatile\s*\(", text):
            depth, i, quoted = 1, m.end(), False
            while depth:
                c = text[i]
                if c == '"' and text[i - 1] != "\\":
                    quoted = not quoted
                elif not quoted:
                    depth += (c == "(") - (c == ")")
                i += 1
            s = text[m.end():i]
            if "{m0}" in s:
                yield name, s


def test_every_copy_waits_for_its_operands():
    found = list(statements())
    assert {name for name, _ in found} >= {"lds_dma.hpp", "packed.hip"} and len(found) >= 3
    for name, s in found:
        first = re.match(r'\s*"s_nop (\d+)\\n\\t', s)
        assert first and int(first[1]) >= 4, (name, s)
