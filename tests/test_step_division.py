"""A row's cut by division (mako_amd/csrc/k_step_cut.hip), its workgroup's lanes one after the other on the CPU."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def test_mass_at_a_bins_end(tmp_path):
    exe = str(tmp_path / "step_division_test")
    subprocess.run(["amdclang++", "-x", "c++", "-std=c++17", "-O1", "-ffp-contract=off", "-Wall", "-I", os.path.join(HERE, "cpu", "lanes"),
                    os.path.join(HERE, "cpu", "step_division_test.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout + r.stderr
