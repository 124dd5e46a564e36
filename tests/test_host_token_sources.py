"""What the token operators' sources promise and no run can show."""

from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "nnunet-mlx_amd" / "csrc"


def _arguments(text: str, at: int) -> list[str]:
    """The arguments of the call whose opening parenthesis is at ``at``."""
    depth, start, found = 0, at + 1, []
    for i in range(at, len(text)):
        if text[i] in "([{":
            depth += 1
        elif text[i] in ")]}":
            depth -= 1
            if depth == 0:
                return found + [text[start:i].strip()]
        elif text[i] == "," and depth == 1:
            found.append(text[start:i].strip())
            start = i + 1
    raise AssertionError("unbalanced call")


@pytest.mark.parametrize("name", ["nnx_blocks.hip", "nnx_blocktile.h", "nnx_tokens.hip"])
def test_bounds_checked_offsets(name):
    """A buffer access is checked by its lane's offset alone: nothing may stand in the scalar one."""
    text = (CSRC / name).read_text()
    for match in re.finditer(r"__builtin_amdgcn_raw_buffer_(load|store)_\w+\(", text):
        arguments = _arguments(text, match.end() - 1)
        assert arguments[-2] == "0", (match.group(), arguments)
