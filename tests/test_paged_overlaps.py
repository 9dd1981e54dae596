"""The paged operators refuse arguments that share memory where a call writes, without a GPU: on the stand-in HIP runtime, in a child process (tests/paged_overlap_case.py)."""
import os
import shutil
import subprocess
import sys

import pytest
import torch

HERE = os.path.dirname(os.path.abspath(__file__))


def run_case(script, tmp_path):
    if torch.cuda.is_available():
        pytest.skip("a real GPU is present: the stand-in runtime is for machines without one")
    if not shutil.which("g++") or not os.path.exists("/opt/rocm/include/hip/hip_runtime_api.h"):
        pytest.skip("needs g++ and the HIP headers to build the stand-in runtime")
    fake = str(tmp_path / "libfakehip.so")
    subprocess.check_call(["g++", "-O1", "-shared", "-fPIC", "-w", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-o", fake, os.path.join(HERE, "fake_hip", "fake_hip.cpp")])
    p = subprocess.run([sys.executable, os.path.join(HERE, script)], capture_output=True, text=True, timeout=300, env=dict(os.environ, LD_PRELOAD=fake))
    assert p.returncode == 0, (p.returncode, p.stdout[-500:], p.stderr[-3000:])
    return p.stdout


def test_written_arguments_share_no_memory_with_others(tmp_path):
    out = run_case("paged_overlap_case.py", tmp_path)
    assert int(out.split("overlaps ok")[1]) >= 90


def test_caches_that_are_written_share_no_rows(tmp_path):
    accepted, refused = (int(x) for x in run_case("paged_kv_case.py", tmp_path).split("kv ok")[1].split())
    assert accepted >= 9 and refused >= 80
