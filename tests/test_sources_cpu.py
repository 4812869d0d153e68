"""Rules of the CUDA sources that no run can show reliably, read from the sources."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "roofline_decoding_b200" / "csrc"
SOURCES = sorted([*CSRC.glob("*.cu"), *CSRC.glob("*.cuh")])


def asm_statements(text):
    """The text of every asm statement, by its balanced parentheses."""
    for m in re.finditer(r"\basm\b(?:\s+volatile)?\s*\(", text):
        depth, i, quoted = 1, m.end(), False
        while depth:
            c = text[i]
            if c == '"' and text[i - 1] != "\\":
                quoted = not quoted
            elif not quoted:
                depth += (c == "(") - (c == ")")
            i += 1
        yield text[m.start():i]


def test_loads_from_tensor_memory_wait_in_their_own_statement():
    """tcgen05.ld writes its registers later; only a wait in the same statement keeps the
    compiler from using, moving or spilling them before they are there."""
    seen = 0
    for path in SOURCES:
        for s in asm_statements(path.read_text()):
            if "tcgen05.ld." in s:
                seen += 1
                assert "tcgen05.wait::ld" in s, f"{path.name}: {s[:120]}"
    assert seen > 0
