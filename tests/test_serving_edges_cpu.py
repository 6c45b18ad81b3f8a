"""The serving operators without a GPU: what the host decides at their edges."""
import os
import re

import flash_colreduce_b200 as fc

CSRC = os.path.join(os.path.dirname(fc.__file__), "csrc")


def status_codes():
    """Every kernel's status codes as the sources define them: [(name, code)]."""
    found = []
    for name in sorted(os.listdir(CSRC)):
        with open(os.path.join(CSRC, name)) as f:
            found += [(n, int(c)) for n, c in re.findall(r"\b(ST_[A-Z0-9_]+)\s*=\s*(\d+)", f.read())]
    return found


def test_a_status_code_names_one_wait():
    """All kernels of a device report into one mailbox: a code must say which kernel and which wait it was."""
    found = status_codes()
    assert len(found) > 50 and len({n for n, _ in found}) == len(found)
    codes = {}
    for name, code in found:
        codes.setdefault(code, []).append(name)
    assert {c: n for c, n in codes.items() if len(n) > 1} == {}
