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


def _body(text: str, opening: str) -> str:
    at = text.index(opening)
    depth = 0
    for i in range(text.index("{", at), len(text)):
        depth += (text[i] == "{") - (text[i] == "}")
        if depth == 0:
            return text[at:i]
    raise AssertionError("unbalanced body")


def test_lanes_that_exchange_through_lds():
    """What lanes of one wave leave for each other in LDS is fenced off on both sides."""
    flush = _body((CSRC / "nnx_blocktile.h").read_text(), "void flush(int pass) const {")
    assert flush.index("wave_sync()") < flush.index("*(const u32x4*)") < flush.rindex("wave_sync()")
    packing = _body((CSRC / "nnx_blocks.hip").read_text(), "if (over <= room) {")
    write, read = packing.index("spare[to] = y"), packing.index("in ? spare[")
    assert packing.index("wave_sync()") < write < packing.rindex("wave_sync()") < read


@pytest.mark.parametrize("name", ["block_select_workspace", "block_attention_workspace"])
def test_no_exception_leaves_a_size_query(name):
    """Refusals are built as strings, which may fail to be allocated: everything is caught."""
    body = _body((CSRC / "nnx_blocks.hip").read_text(), f"size_t {name}(")
    assert "catch (...)" in body
