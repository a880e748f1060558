"""What the selective scan's and the short convolution's sources and entry points keep to, without a GPU."""

import re
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "rnn_with_grm_amd" / "csrc"


def calls(text, name):
    """The argument lists of the calls of `name` in a source."""
    for m in re.finditer(name + r"\(", text):
        args, depth = [""], 0
        for ch in text[m.end():]:
            if ch == "," and depth == 0:
                args.append("")
                continue
            depth += (ch in "([{") - (ch in ")]}")
            if depth < 0:
                break
            args[-1] += ch
        yield [x.strip() for x in args]


def test_masked_loads_have_no_scalar_offset():
    """Rows past a tile's end read zeros because their offset lies outside the buffer resource.  That holds for the
    vector register's part of an offset; a scalar one need not be in the range check."""
    found = [c for p in sorted(CSRC.glob("selective*")) for c in calls(p.read_text(), r"__builtin_amdgcn_raw_buffer_load_\w+")]
    assert len(found) >= 5 and all(len(c) == 4 for c in found)
    assert [c for c in found if c[2] != "0"] == []
