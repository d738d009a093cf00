"""The header's constants under the same names in Python."""
import os
import re

from sejong_amd import _native as N

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_constants_of_the_header():
    with open(os.path.join(ROOT, "include", "sejong_hip.h")) as f:
        found = re.findall(r"^#define (SJ_\w+) (\d+)\b", f.read(), re.M)
    names = {name: int(value) for name, value in found if name != "SJ_OK" and not name.startswith("SJ_ERR_")}
    assert {"SJ_BF16", "SJ_PLAN_ROWS", "SJ_FORK_LIST_FULL", "SJ_BEAM_MAX"} <= set(names)
    for name, value in names.items():
        assert getattr(N, name) == value, name
