"""What the attention operators' host side does with its workspace, streams and errors, without a GPU: the library's host
sources are compiled against a CUDA runtime and kernels that record their calls (tests/attention_host_check.cpp)."""

import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "voxwerk_b200", "csrc")


@pytest.fixture(scope="module")
def checker(tmp_path_factory):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc))), "include")
    exe = str(tmp_path_factory.mktemp("host") / "attention_host_check")
    sources = [os.path.join(ROOT, "tests", "attention_host_check.cpp"), os.path.join(CSRC, "vw_api.cpp"),
               os.path.join(CSRC, "vw_attention.cpp")]
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", cuda, "-I", CSRC, "-I", os.path.join(ROOT, "include"), *sources,
                    "-o", exe], check=True)
    return exe


SCENARIOS = ["captured_workspace", "outgrown_workspace", "growth_under_capture", "captured_sampler",
             "error_on_another_stream", "error_of_an_enqueued_call", "workspace_order"]


@pytest.mark.parametrize("scenario", SCENARIOS)
def test_host_side(checker, scenario):
    run = subprocess.run([checker, scenario], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0, run.stdout + run.stderr
