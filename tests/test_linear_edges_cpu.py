"""Inputs of the linear attention, its step and the gated norm that few calls have, on CPU tensors, and the kernels' addresses on the host."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_row_addresses(tmp_path):
    exe = str(tmp_path / "check")
    subprocess.run(["g++", "-O2", "-std=c++17", "-I", os.path.join(ROOT, "pope-pytorch_amd", "csrc"), os.path.join(ROOT, "tests", "linear_rows_check.cpp"),
                    "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout
