"""How paged attention cuts a call's rows into pieces (csrc/paged.h, compiled for the host): no row is lost.  CPU only."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_every_row_is_computed_and_joined(tmp_path):
    exe = str(tmp_path / "paged_cut")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", os.path.join(ROOT, "tests", "paged_cut.cpp"), "-o", exe], check=True)
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout == "ok\n", out.stdout + out.stderr
