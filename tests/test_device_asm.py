"""Hazards that the compiler does not see inside inline assembly, looked for in the sources (no GPU)."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "valkyr_amd", "csrc")


def statements():
    """(file, its inline assembly statements, each a list of instructions)."""
    for path in sorted(glob.glob(os.path.join(CSRC, "*.h*"))):
        text = open(path).read()
        for m in re.finditer(r"\basm\s*(?:volatile)?\s*\(\s*((?:\"(?:[^\"\\]|\\.)*\"\s*)+)", text):
            body = "".join(re.findall(r"\"((?:[^\"\\]|\\.)*)\"", m.group(1)))
            yield os.path.basename(path), [x.strip() for x in re.split(r"\\n|\\t|;", body) if x.strip()]


def test_loads_to_lds_wait_for_their_address():
    """A load to LDS takes its address from M0 and needs one wait state after a scalar write of it."""
    loads = 0
    for name, ops in statements():
        for i, op in enumerate(ops):
            if not re.search(r"\blds$", op):
                continue
            loads += 1
            assert i >= 2 and ops[i - 1].startswith("s_nop") and re.match(r"s_mov_b32 m0\b", ops[i - 2]), (name, ops)
    assert loads >= 2
