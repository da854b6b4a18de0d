"""Inputs of the linear attention, its step and the gated norm that few calls have, on CPU tensors, and the kernels' addresses on the host."""
import math
import os
import subprocess

import pytest
import torch

import pope_amd
from linear_common import Case, run

CPU = torch.device("cpu")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_row_addresses(tmp_path):
    exe = str(tmp_path / "check")
    subprocess.run(["g++", "-O2", "-std=c++17", "-I", os.path.join(ROOT, "pope-pytorch_amd", "csrc"), os.path.join(ROOT, "tests", "linear_rows_check.cpp"),
                    "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan, "lowest"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masked_rows_reach_no_gradient(dtype, value):
    case = Case(CPU, B=2, N=150, mask="empty", dtype=dtype, initial=True)
    clean = run(pope_amd, case)
    x = torch.finfo(dtype).min if value == "lowest" else value
    case.k, case.v = (t.masked_fill(~case.mask[:, None, :, None], x) for t in (case.k, case.v))
    got = run(pope_amd, case)
    for n in clean:
        assert torch.equal(got[n], clean[n]), n
    assert not got["d_k"][0].any() and not got["d_v"][0].any()
