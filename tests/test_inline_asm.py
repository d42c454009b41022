"""Inline assembly in the kernels: the compiler places no wait states inside it."""
import glob
import os
import re

from ferrisinfer_amd import build

CSRC = os.path.join(os.path.dirname(build.__file__), "csrc")


def statements():
    for path in sorted(glob.glob(os.path.join(CSRC, "**", "*.h*"), recursive=True)):
        with open(path) as f:
            text = f.read()
        for at in re.finditer(r"\basm\b[^(;]*\(", text):
            code = re.match(r"\s*((?:\"(?:[^\"\\]|\\.)*\"\s*)+)", text[at.end():])
            if code:
                joined = "".join(re.findall(r"\"((?:[^\"\\]|\\.)*)\"", code.group(1)))
                yield os.path.basename(path), [s for s in re.split(r"\\n|\\t|;", joined) if s.strip()]


def test_a_load_to_lds_waits_a_state_for_m0():
    """A load to LDS takes its address from m0, which needs a wait state behind a scalar write of it."""
    found = 0
    for name, code in statements():
        for i, instruction in enumerate(code):
            if re.match(r"\s*s_\w+\s+m0\b", instruction):
                found += 1
                assert re.match(r"\s*s_nop\b", code[i + 1]), (name, code)
            elif "_lds" in instruction:
                assert i > 0 and any("s_nop" in c for c in code[:i]), (name, code)  # m0 is set in the same statement
    assert found > 0
