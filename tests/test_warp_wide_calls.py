"""No warp-wide exchange with a full mask inside a conditional expression (no GPU needed).

`lane < k ? f(__shfl_sync(0xffffffffu, v, 0)) : 0` calls the shuffle in some lanes only, and a shuffle whose mask names all lanes waits for the others
for good. Statements are cut at semicolons and braces; inside one, an exchange is in a branch of a conditional expression when a
`?` stands before it in one of the groups (parentheses, brackets) that enclose it, with no comma of that group between them.
"""

import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "drama_rs_b200", "csrc")
CALL = re.compile(r"(__shfl_\w*sync|__ballot_sync|__reduce_\w+_sync|__match_any_sync|warp_sum|warp_max)\(")


def conditional_exchanges(text: str) -> list[str]:
    text = re.sub(r"//[^\n]*|/\*.*?\*/|\"(\\.|[^\"\\])*\"", "", text, flags=re.S)
    found = []
    for statement in re.split(r"[;{}]", text):
        open_groups = [False]  # per enclosing group: a `?` has been seen
        i = 0
        while i < len(statement):
            m = CALL.match(statement, i)
            if m and (i == 0 or not (statement[i - 1].isalnum() or statement[i - 1] == "_")):
                if any(open_groups):
                    found.append(" ".join(statement.split()))
                i = m.end() - 1
            c = statement[i]
            if c in "([":
                open_groups.append(False)
            elif c in ")]" and len(open_groups) > 1:
                open_groups.pop()
            elif c == "?":
                # a template constant against a number is decided by the compiler
                open_groups[-1] = not re.search(r"\b[A-Z][A-Z0-9_]* == \d+ $", statement[:i])
            elif c == ",":
                open_groups[-1] = False
            i += 1
    return found


def test_the_scan_tells_them_apart():
    assert conditional_exchanges("float e = lane < k ? expf(v - __shfl_sync(0xffffffffu, v, 0)) : 0.f;")
    assert conditional_exchanges("x = a ? 1.f : warp_sum(v);")
    assert not conditional_exchanges("s = (hi ? a : b) + __shfl_xor_sync(0xffffffffu, hi ? b : a, 16);")
    assert not conditional_exchanges("u = GEMM == 0 ? __shfl_sync(0xffffffffu, v, 1) : s;")
    assert not conditional_exchanges("const float t = c ? a : b, s = warp_sum(v);")


@pytest.mark.parametrize("name", sorted(f for f in os.listdir(CSRC) if f.endswith((".cuh", ".cu"))))
def test_exchanges_are_not_conditional(name):
    assert conditional_exchanges(open(os.path.join(CSRC, name)).read()) == []
