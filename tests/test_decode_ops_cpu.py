"""The text-decoder operators' C entries refuse bad arguments before they touch a GPU."""
from __future__ import annotations

import pytest

P = 1 << 20  # a 16-byte aligned address that no call reads


@pytest.fixture(scope="module")
def lib(pkg):
    from gemma4_omni_b200 import _lib, build
    build.build_library()
    return _lib.load()


def refused(lib, name, good, changes):
    """Every change to the argument list is refused as an invalid argument."""
    for at, value in changes:
        args = list(good)
        args[at] = value
        assert getattr(lib, name)(*args) == -1, (name, at, value)


def test_plan_entries(lib):
    plan = [1, P, P, 4, 2, 4, 16, P, P, P, 8, P, P, P, P, P, P, P, None]
    refused(lib, "lb_plan_pages", plan, [(0, 0), (0, 8193), (1, None), (3, 0), (3, 262145), (4, 0), (5, 0), (6, 8), (6, 24),
                                         (6, 512), (9, None), (10, 0), (10, 1 << 27), (14, None), (17, None)])
    refused(lib, "lb_commit_pages", [1, P, 4, 2, 4, 16, P, P, P, P, P, P, None], [(0, 0), (6, None), (8, None), (11, None)])
    refused(lib, "lb_release_pages", [1, P, 4, 2, 4, 16, P, P, P, P, None], [(0, 0), (1, None), (9, None)])


def test_append_entry(lib):
    good = [P, 64, 64, P, 64, 64, 1, 2, 1, 64, P, P, P, P, P, 4, 16, None, None]
    refused(lib, "lb_op_kv8_append", good, [(0, None), (6, 2), (6, 7), (7, 0), (8, 0), (9, 24), (9, 1024), (10, None),
                                            (11, P + 8), (15, 0), (16, 20), (16, 512)])


def test_attention_entry(lib):
    good = [P, 64, 64, 1, 1, 1, 4, 2, 64, P, P, P, P, 4, 16, P, 2, P, P, 1, 0.1, 0, 0.0, P, None, None, P, None]
    refused(lib, "lb_op_kv8_attention", good, [(0, None), (3, 0), (3, 2), (4, 0), (5, 0), (7, 3), (8, 96), (9, P + 4), (13, 0),
                                               (14, 8), (15, None), (16, 0), (19, 0), (21, -1), (22, -1.0),
                                               (22, float("nan")), (23, None), (26, None), (26, P + 4)])
    assert lib.lb_kv8_attention_workspace(96, 4, 2, 1) == -1 and lib.lb_kv8_attention_workspace(64, 3, 2, 1) == -1
    assert 0 < lib.lb_kv8_attention_workspace(128, 4, 2, 1) < lib.lb_kv8_attention_workspace(128, 4, 2, 100)


def test_norm_entry(lib):
    good = [P, 64, P, 64, 1, P, 0, 1, 64, 1e-6, 0, 4, P, P, P, None]
    refused(lib, "lb_op_rms_norm8", good, [(0, None), (1, 63), (3, 60), (4, 2), (6, 3), (7, 0), (8, 0), (8, 16385), (10, -1),
                                           (10, 48), (11, 1), (12, None), (13, None)])


def test_w4_entry(lib):
    good = [P, 128, 1, None, 0, 1, P, P, 128, 64, 128, P, 64, 1, None]
    refused(lib, "lb_op_w4_matvec", good, [(0, None), (1, 64), (2, 0), (2, 4), (3, P), (4, 128), (5, 0), (6, P + 1), (8, 16),
                                           (8, 256), (9, 0), (10, 100), (12, 63), (13, 2)])


def test_wrappers_have_no_cpu_path(pkg):
    import torch
    from gemma4_omni_b200 import decode_ops as ops
    with pytest.raises(ValueError):
        ops.rms_norm8(torch.zeros(2, 64), torch.ones(64))
    with pytest.raises(ValueError):
        ops.Int4Weight(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.float16))
    with pytest.raises(ValueError):
        ops.PageDirectory.create(sessions=2, max_pages=2, pages=4, page_tokens=16, device="cpu")
