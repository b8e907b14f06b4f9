"""The step's entry points where launches fail, without a GPU."""
import os
import subprocess

from mako_amd import api

HERE = os.path.dirname(os.path.abspath(__file__))


def test_errors_of_launches(tmp_path):
    exe = str(tmp_path / "step_launch_test")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-O1", "-rdynamic", os.path.join(HERE, "cpu", "step_launch_test.cpp"), "-o", exe, "-ldl"], check=True)
    r = subprocess.run([exe, api.LIB_PATH], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout + r.stderr
