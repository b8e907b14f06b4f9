"""include/mako_step.h without a GPU: exports, layouts, and what the entry points refuse."""
import ctypes
import os
import re
import subprocess

from mako_amd import api, step

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_exports_match_header():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "mako_step.h")).read(), flags=re.S)
    names = set(re.findall(r"\b(mako_step_\w+)\s*\(", text))
    assert names == set(step.EXPORTS)
    lib = step.load()
    for n in names:
        assert hasattr(lib, n), n


def test_layouts(tmp_path):
    """The descriptors' sizes and offsets as a C compiler has them."""
    assert step.CUT_DTYPE.itemsize == 32
    fields = {"mako_cut_desc": step.CutDesc, "mako_verify_desc": step.VerifyDesc, "mako_blocks_desc": step.BlocksDesc}
    lines = ['#include <stddef.h>', '#include <stdio.h>', '#include "mako_step.h"', "int main(void) {"]
    for c, py in fields.items():
        lines.append('printf("%%zu\\n", sizeof(%s));' % c)
        lines += ['printf("%%zu\\n", offsetof(%s, %s));' % (c, f[0]) for f in py._fields_]
    lines += ['printf("%%zu\\n", offsetof(mako_row_cut, %s));' % f for f in step.CUT_DTYPE.names]
    lines.append("return 0; }")
    exe = str(tmp_path / "layout")
    subprocess.run(["gcc", "-x", "c", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), "-", "-o", exe], input="\n".join(lines), text=True, check=True)
    got = [int(x) for x in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for py in fields.values():
        want += [ctypes.sizeof(py)] + [getattr(py, f[0]).offset for f in py._fields_]
    want += [step.CUT_DTYPE.fields[f][1] for f in step.CUT_DTYPE.names]
    assert got == want


def test_refusals_without_a_context():
    lib = step.load()
    p = ctypes.c_void_p()
    for rows, vocab in ((0, 8), (8, 0), (step.MAX_ROWS + 1, 8), (8, step.MAX_VOCAB + 1)):
        assert lib.mako_step_create(ctypes.byref(p), 0, rows, vocab) == api.MAKO_ERR_INVALID_ARG
        assert not p.value
    assert lib.mako_step_create(None, 0, 1, 1) == api.MAKO_ERR_INVALID_ARG
    assert lib.mako_step_last_error(None) == b"null context"
    for name, desc in (("cut_rows", step.CutDesc()), ("verify_drafts", step.VerifyDesc()), ("assign_blocks", step.BlocksDesc())):
        assert getattr(lib, "mako_step_" + name)(None, ctypes.byref(desc), None) == api.MAKO_ERR_INVALID_ARG
    lib.mako_step_destroy(None)


def test_refused_calls(tmp_path):
    exe = str(tmp_path / "step_checks_test")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-O1", os.path.join(ROOT, "tests", "cpu", "step_checks_test.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout
