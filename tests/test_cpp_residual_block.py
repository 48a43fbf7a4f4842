"""Runs the C++ program of the operators for sequences
(tests/cpp/gpu_residual_block_test.cpp, built by __graft_entry__.build())."""
import subprocess

import pytest

from test_cpp_api import _exe


def _run(*args):
    out = subprocess.run([_exe("gpu_residual_block_test"), *args],
                         stdout=subprocess.PIPE, stderr=subprocess.STDOUT,
                         text=True, timeout=120)
    assert out.returncode == 0, out.stdout[-4000:]
    assert "0 failures" in out.stdout


def test_refusals():
    _run("--host")


@pytest.mark.gpu
def test_operators_and_gradients():
    _run()
