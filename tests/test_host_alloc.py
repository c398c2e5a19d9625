"""The library's host code when memory runs out or calls are refused, on a HIP runtime of host memory
(cpp/fake_hip.cpp, fake_device.py): a failed allocation leaves a handle that later calls can use."""
import os
import subprocess
import sys

import pytest

import nanovllm_moe

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("fake") / "libfake_hip.so")
    build = subprocess.run(["g++", "-O1", "-std=c++17", "-fPIC", "-shared", os.path.join(HERE, "cpp", "fake_hip.cpp"), "-o", so],
                           stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert build.returncode == 0, build.stdout
    return so


def _run(fake, check):
    run = subprocess.run([sys.executable, os.path.join(HERE, "fake_device.py"), fake, nanovllm_moe.LIB_PATH, check],
                         stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    assert run.returncode == 0 and run.stdout.strip().endswith("ok"), run.stdout


def test_weights(fake):
    """Storing weights: all buffers or none, whichever allocation fails."""
    _run(fake, "weights")


def test_workspace(fake):
    """A call that cannot grow the workspace: the next, smaller one finds one that fits it, not parts of two."""
    _run(fake, "workspace")


def test_picks(fake):
    """The buffer of a call's router picks after a failed growth."""
    _run(fake, "picks")


def test_refused(fake):
    """A call behind a router that is refused allocates, launches and waits for nothing."""
    _run(fake, "refused")


def test_clears(fake):
    """New buffers are clear before the caller's stream, which may not wait for the default one, stores into them."""
    _run(fake, "clears")


def test_mx_workspace(fake):
    """An MXFP4 handle's workspace holds what its kernels use, and calls without allocation take what fits."""
    _run(fake, "mx_workspace")


def test_hybrid_leaves_nothing(fake):
    """The offload executor's handle gives back every allocation, those of its store call too."""
    _run(fake, "hybrid_leaves_nothing")


def test_hybrid_staging(fake):
    """The executor's staging buffers after a call that could not grow them."""
    _run(fake, "hybrid_staging")
