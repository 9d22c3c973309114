"""Host code around launches, compiled with the runtime's calls replaced by ones that a test can look into (launch_host.cu)."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "yamoe_b200", "csrc")


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    out = str(tmp_path_factory.mktemp("launch") / "launch_host")
    build = subprocess.run([nvcc, "-std=c++17", "-O1", "-gencode", "arch=compute_100a,code=sm_100a", "--expt-relaxed-constexpr", "-I", CSRC, "-o", out,
                            os.path.join(HERE, "launch_host.cu"), "-ldl"], capture_output=True, text=True, timeout=600)
    assert build.returncode == 0, build.stderr
    return out


def check(program, name):
    run = subprocess.run([program, name], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0, run.stdout + run.stderr


def test_shared_memory_asked_for_by_two_threads(program):
    """A size that one thread has set and remembers is not made smaller by another that had asked for less."""
    check(program, "threads")


def test_refused_calls_leave_no_error_behind(program):
    """The runtime keeps the error of a launch, an attribute or a memset that it refused; the next launch would be taken for the one that failed."""
    check(program, "refused")


@pytest.mark.parametrize("name", ["tiles", "parts", "ring"])
def test_arithmetic_that_kernels_and_launchers_share(program, name):
    """The functions themselves, over all sizes that they may meet."""
    check(program, name)
