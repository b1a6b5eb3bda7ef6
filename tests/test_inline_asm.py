"""What the kernels' inline assembly declares."""
from __future__ import annotations

import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "turborag_amd" / "csrc"


def test_registers_written_by_name_are_clobbers():
    """m0, vcc and exec as a destination in an asm statement: named among its clobbers."""
    seen = 0
    for path in sorted(CSRC.glob("*.h*")):
        for stmt in re.findall(r"\basm\b(?:\s+volatile)?\s*\((.*?)\);", path.read_text(), re.S):
            text = "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', stmt))
            for reg in re.findall(r"(?:^|\\n\\t|;)\s*s_\w+ (m0|vcc|exec)\b", text):
                seen += 1
                clobbers = stmt.rsplit(":", 1)[-1]
                assert f'"{reg}"' in clobbers, f"{path.name}: asm writes {reg} and does not say so"
    assert seen
