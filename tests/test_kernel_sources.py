"""What the kernel sources must not contain, checked on their text."""

import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rustllm_amd",
                    "csrc")


def inline_assembly():
    for path in sorted(glob.glob(os.path.join(CSRC, "*.h*"))):
        with open(path) as f:
            text = re.sub(r"//[^\n]*", "", f.read())
        for m in re.finditer(r"\basm\b(?:\s+volatile)?\s*\(", text):
            depth, end = 1, m.end()
            while depth:
                depth += {"(": 1, ")": -1}.get(text[end], 0)
                end += 1
            body = text[m.end():end - 1]
            yield os.path.basename(path), "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', body))


def test_no_vector_alu_instruction_in_inline_assembly():
    """The compiler adds the wait states between a matrix product and a vector
    instruction that reads its result (12 for a 32 x 32 x 16 product), and the other
    hazards' too, for its own instructions only."""
    found = list(inline_assembly())
    assert found  # the loads to LDS
    for name, code in found:
        assert not re.search(r"\bv_[a-z0-9_]+", code), (name, code)
