"""Scratch memory of the step's kernels: none (what it costs: tests/test_kernel_scratch.py), but 12 bytes of the fp32 kernel for wide
cuts, which holds a row's division and a second try beside the common way."""
import os

import pytest

from mako_amd import api
from test_kernel_scratch import _code_objects, _kernels

STEP = "_ZN4mako4step"
ALLOWED = {"wide_kernelINS0_3F32E": 12}


def test_scratch_memory():
    if not os.path.exists(api.LIB_PATH):
        pytest.skip("the library is not built")
    with open(api.LIB_PATH, "rb") as f:
        data = f.read()
    found = {}
    for elf in _code_objects(data):
        found.update({k: v for k, v in _kernels(elf).items() if k.startswith(STEP)})
    for kernel, count in (("scan_kernel", 3), ("row_kernel", 3), ("look_kernel", 3), ("wide_kernel", 3), ("probs_kernel", 3), ("left_kernel", 9), ("draw_kernel", 9),
                          ("blocks_kernel", 1), ("counts_kernel", 1), ("plan_kernel", 1), ("apply_kernel", 1)):
        assert sum(kernel in k for k in found) == count, (kernel, sorted(found))
    most = {k: next((v for part, v in ALLOWED.items() if part in k), 0) for k in found}
    assert not {k: v for k, v in found.items() if v > most[k]}
