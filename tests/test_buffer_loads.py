"""Buffer loads that count on the end of their resource carry their whole offset in the lane
operand, the one that the end is specified to be compared with (no GPU).

The scalar offset is for loads whose resource is empty or ends behind everything they reach.
"""
from __future__ import annotations

import re

from conftest import PKG_DIR

# (file, scalar offset) of the loads of that kind: a resource of no bytes, or of 2^31.
UNBOUNDED = {
    ("pa_tiles.h", "uoff"),  # load_tile
    ("pa_decode_linear.hip", "(j & 1) * 16 * (int)a.ldw + pair * 64"),  # past the end by the lane's offset
    ("pa_decode_linear.hip", "u * (XPACK ? 1024 : 64)"),
    ("pa_decode_linear.hip", "u * 1024"),
    ("pa_decode_linear.hip", "u * 64"),
}
# Which operand is the scalar offset.
CALLS = {"raw_buffer_load": 2, "raw_buffer_store": 3, "raw_ptr_buffer_load_lds": 4}


def arguments(text, at):
    """The top-level arguments of the call whose opening bracket is at `at`."""
    depth, start, out = 0, at + 1, []
    for i in range(at, len(text)):
        depth += text[i] in "([{"
        depth -= text[i] in ")]}"
        if depth == 0 or depth == 1 and text[i] == ",":
            out.append(" ".join(text[start:i].split()))
            start = i + 1
        if depth == 0:
            return out
    raise AssertionError("unbalanced call")


def test_scalar_offsets():
    found = set()
    for path in sorted((PKG_DIR / "csrc").iterdir()):
        text = path.read_text()
        for m in re.finditer(r"__builtin_amdgcn_(raw_\w+?)(?:_b\d+)?\(", text):
            offset = arguments(text, m.end() - 1)[CALLS[m.group(1)]]
            if offset != "0":
                found.add((path.name, offset))
    assert found == UNBOUNDED
