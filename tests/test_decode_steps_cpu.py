"""The entries that plan and commit a step, and attention's numbers, refuse bad arguments before they touch a GPU."""
from __future__ import annotations

import math

import pytest

P = 1 << 20  # a 16-byte aligned address that no call reads


@pytest.fixture(scope="module")
def lib(pkg):
    from gemma4_omni_b200 import _lib, build
    build.build_library()
    return _lib.load()


@pytest.mark.parametrize("name,good,changes", [
    ("lb_plan_step", [1, P, P, 4, 2, 4, 16, P, P, P, 8, P, P, P, P, P, P, P, P, None],
     [(0, 0), (0, 8193), (1, None), (3, 0), (3, 262145), (4, 0), (5, 0), (6, 8), (6, 512), (9, None), (10, 0), (10, 1 << 27), (14, None), (18, None)]),
    ("lb_commit_step", [1, P, 4, 2, 4, 16, P, P, P, P, P, P, P, None],
     [(0, 0), (1, None), (2, 0), (5, 24), (6, None), (7, None), (9, None), (10, None), (12, None)]),
    ("lb_op_kv8_attention", [P, 64, 64, 1, 1, 1, 4, 2, 64, P, P, P, P, 4, 16, P, 2, P, P, 1, 0.1, 0, 0.0, P, None, None, P, None],
     [(22, math.inf), (22, math.nan), (22, -0.5)]),
])
def test_refusals(lib, name, good, changes):
    for at, value in changes:
        args = list(good)
        args[at] = value
        assert getattr(lib, name)(*args) == -1, (at, value)
