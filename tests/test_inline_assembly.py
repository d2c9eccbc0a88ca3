"""Memory accesses in inline assembly: the waits that the instruction set wants of the program are part of the text.

The compiler keeps five states between an instruction of the vector unit that writes a scalar register (v_readfirstlane, or v_readlane of a spilled one) and a memory
access that reads it, but it does not see that a statement of text is such an access.  So the text has them itself: five states in front of the access, or the
register copied by the scalar unit, which waits for the vector unit by itself and which an access may follow at once.  m0 is set a state or more in front of an access
to LDS.
"""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "stk_amd", "csrc")
ACCESS = re.compile(r"(buffer|global|flat|scratch)_(load|store|atomic)")


def _statements():
    """(where, instructions, operands' constraints in their order) of every asm statement."""
    for name in sorted(os.listdir(CSRC)):
        if not name.endswith((".h", ".hip")):
            continue
        text = open(os.path.join(CSRC, name)).read()
        macros = dict(re.findall(r"^#define (STK_\w+) (.*)$", text, re.M))
        for at in re.finditer(r"\basm\s*(?:volatile\s*)?\(", text):
            depth, end, quoted = 1, at.end(), False
            while depth:
                c = text[end]
                if c == '"' and text[end - 1] != "\\":
                    quoted = not quoted
                depth += 0 if quoted else (c == "(") - (c == ")")
                end += 1
            body = text[at.end():end - 1]
            for _ in range(2):
                body = re.sub(r"\bSTK_\w+", lambda m: macros.get(m.group(0), m.group(0)), body)
            parts, depth, quoted, last = [], 0, False, 0
            for i, c in enumerate(body):   # template : outputs : inputs : clobbers
                if c == '"' and body[i - 1] != "\\":
                    quoted = not quoted
                if quoted:
                    continue
                depth += (c in "([") - (c in ")]")
                if c == ":" and not depth and body[i - 1:i + 2].count(":") == 1:
                    parts.append(body[last:i])
                    last = i + 1
            parts.append(body[last:])
            template = "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', parts[0])).replace("\\t", "").split("\\n")
            constraints = [c for part in parts[1:3] for c in re.findall(r'"([^"]*)"\s*\(', part)]
            yield f"{name}:{text.count(chr(10), 0, at.start()) + 1}", [i.strip() for i in template if i.strip()], constraints


ALL = list(_statements())


def _states(instruction):
    nop = re.match(r"s_nop (\d+)", instruction)
    return int(nop.group(1)) + 1 if nop else 1


def test_statements_are_found():
    assert sum(any(ACCESS.match(i) for i in text) for _, text, _ in ALL) >= 9


@pytest.mark.parametrize("where,text,constraints", [s for s in ALL if any(ACCESS.match(i) for i in s[1])], ids=lambda v: v if isinstance(v, str) else "")
def test_waits_in_front_of_accesses(where, text, constraints):
    copied, m0 = set(), None    # operands that the scalar unit wrote here; states since m0 was written
    states = 0
    for i in text:
        used = [int(n) for n in re.findall(r"%(\d+)", i)]
        if ACCESS.match(i):
            for n in used:
                assert constraints[n].strip("=+&") != "s" or n in copied or states >= 5, f"{where}: {i} reads %{n} {states} states into the statement"
            assert not i.endswith("lds") and " lds" not in i and "_lds_" not in i or m0 is not None and m0 >= 1, f"{where}: m0"
        if re.match(r"s_mov_b", i) and used and constraints[used[0]].startswith("=&s"):
            copied.add(used[0])
        states += _states(i)
        if m0 is not None:
            m0 += _states(i)
        if re.match(r"s_\w+ m0,", i):
            m0 = 0
