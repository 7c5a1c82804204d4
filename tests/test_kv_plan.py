"""The paged attention's work plan (csrc/sdq_kv_plan.h), swept on the CPU: tiles, grids
and scratch of any call within their bounds."""
import os
import subprocess

from conftest import PKG, ROOT


def test_every_plan_fits(tmp_path):
    exe = str(tmp_path / "kv_plan")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Wextra", "-I" + os.path.join(PKG, "csrc"),
                    os.path.join(ROOT, "tests", "cpp", "kv_plan.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
