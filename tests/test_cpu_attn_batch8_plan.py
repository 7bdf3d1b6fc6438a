"""How attention of a batch over a cache in 8 bits shares out a step's work between two kernels and their CTAs (csrc/attn_batch_plan.cuh, host and device code): tests/plan/attn_batch8_plan_check.cpp."""
import os
import re
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "qwen_inference_engine_b200", "csrc")
CUDA = os.environ.get("CUDA_HOME") or "/usr/local/cuda"


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    if not shutil.which("g++") or not os.path.exists(os.path.join(CUDA, "include", "cuda_bf16.h")):
        pytest.skip("no C++ compiler or no CUDA headers")
    exe = str(tmp_path_factory.mktemp("plan") / "check8")
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-I", CSRC, "-I", os.path.join(CUDA, "include"), "-o", exe, os.path.join(HERE, "plan", "attn_batch8_plan_check.cpp")])
    return exe


@pytest.mark.parametrize("seed", [1, 2, 3])
def test_every_row_in_one_kernel(check, seed):
    out = subprocess.run([check, str(seed), "300"], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.startswith("ok"), out.stdout
    pieces, cut = map(int, re.findall(r"\d+", out.stdout))
    assert pieces > 10 ** 5 and cut > 10 ** 4, out.stdout
