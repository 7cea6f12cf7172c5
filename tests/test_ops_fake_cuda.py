"""The operators' create and destroy on a made-up CUDA runtime (tests/host/ops_on_fake_cuda.cpp)."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")


@pytest.fixture(scope="module")
def rows(tmp_path_factory):
    """-> (kind, failing call or 0, create's status, copies pending, blocks left, destroy's status, blocks left, wrong frees)"""
    if not shutil.which("g++") or not os.path.exists(os.path.join(CUDA, "include", "cuda_runtime.h")):
        pytest.skip("no C++ compiler or CUDA headers")
    exe = tmp_path_factory.mktemp("fake") / "ops"
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(CUDA, "include"), "-o", str(exe), "-x", "c++",
                    os.path.join(ROOT, "tests", "host", "ops_on_fake_cuda.cpp"), os.path.join(ROOT, "rosenna_b200", "csrc", "ops.cu")], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=60).stdout
    return [tuple(int(v) for v in ln.split()) for ln in out.splitlines()]


def test_weights_have_arrived_when_create_returns(rows):
    """A copy from pageable memory may still be on its way when cudaMemcpy returns, and a run on a stream that does not
    wait for the default one could overtake it."""
    done = [r for r in rows if r[1] == 0]
    assert len(done) == 3 and all(r[2] == 0 and r[3] == 0 for r in done), done


def test_destroy_frees_everything(rows):
    done = [r for r in rows if r[2] == 0]
    assert all(r[5] == 0 and r[6] == 0 and r[7] == 0 for r in done), done


def test_a_failed_create_leaves_nothing(rows):
    """Whichever of its CUDA calls fails."""
    failed = [r for r in rows if r[1] and r[2]]
    assert {r[0] for r in failed} == {0, 1, 2} and all(r[4] == 0 and r[7] == 0 for r in failed), failed
