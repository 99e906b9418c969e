"""What the compiler has to be told about the operators' inline assembly, read in their sources."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "go-metal_amd", "csrc")


def statements(path):
    """(instructions, everything behind them) of each asm statement."""
    text = re.sub(r"//[^\n]*", "", open(path).read())
    for at in re.finditer(r"\basm\s+volatile\s*\(", text):
        depth, end = 1, at.end()
        while depth:
            depth += {"(": 1, ")": -1}.get(text[end], 0)
            end += 1
        body = text[at.end():end - 1]
        code = re.match(r'\s*((?:"(?:[^"\\]|\\.)*"\s*)+)', body)
        yield code.group(1), body[code.end():]


WITH_M0 = re.compile(r"\bm0\s*,|_load_lds_|_lds_dword")      # written, or read: loads into LDS take their address from it


@pytest.mark.parametrize("path", sorted(glob.glob(os.path.join(CSRC, "*"))), ids=os.path.basename)
def test_the_compiler_knows_of_m0(path):
    """As an operand, so that the compiler writes it, or among the registers that are overwritten."""
    for code, rest in statements(path):
        if WITH_M0.search(code):
            assert '"{m0}"' in rest or '"m0"' in rest.split(":")[-1], code


def test_there_is_assembly_to_read():
    assert any(WITH_M0.search(code) for path in glob.glob(os.path.join(CSRC, "*")) for code, _ in statements(path))
