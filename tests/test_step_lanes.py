"""Device functions of the step's kernels on the CPU, a workgroup's lanes one after the other (tests/cpu/lanes)."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def run(tmp_path, name):
    exe = str(tmp_path / name)
    subprocess.run(["amdclang++", "-x", "c++", "-std=c++17", "-O1", "-ffp-contract=off", "-Wall", "-I", os.path.join(HERE, "cpu", "lanes"),
                    os.path.join(HERE, "cpu", name + ".cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout + r.stderr


def test_mass_at_a_bins_end(tmp_path):
    """A row's cut by division (k_step_cut.hip)."""
    run(tmp_path, "step_division_test")


def test_powers_of_two(tmp_path):
    """Weights (step_common.h)."""
    run(tmp_path, "step_exp2_test")
