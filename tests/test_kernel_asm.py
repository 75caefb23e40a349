"""What inline assembly in the kernels' sources promises the compiler: no GPU needed."""
from __future__ import annotations

import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rpgbarenginecuda_amd", "csrc")


def asm_statements():
    for path in sorted(p for ext in ("hip", "h", "cc") for p in glob.glob(os.path.join(CSRC, "*." + ext))):
        text = open(path).read()
        for m in re.finditer(r"\basm(?:\s+volatile)?\s*\(", text):
            depth, at, quoted = 1, m.end(), False
            while depth:
                c = text[at]
                if c == '"':
                    quoted = not quoted
                elif not quoted:
                    depth += {"(": 1, ")": -1}.get(c, 0)
                at += 1
            yield os.path.basename(path), text.count("\n", 0, m.start()) + 1, text[m.end():at - 1]


def test_no_statement_writes_m0():
    """The compiler has uses of its own for M0, and moves or drops its writes of it as if no statement made any: what a
    statement needs there comes in as an operand."""
    found = list(asm_statements())
    assert any('"{m0}"' in body for _, _, body in found)
    assert [(f, line) for f, line, body in found if re.search(r"\bs_\w+ m0,", body)] == []
