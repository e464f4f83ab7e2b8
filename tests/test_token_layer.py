"""The token-model ops of the C++ tl:: layer (host/tests/test_tokens.cpp): tl::layer_norm,
tl::embedding and tl::token_logprobs with their autograd nodes, alone and in one model with
tl::matmul and tl::flash_attention; the exception part needs no GPU."""
import os
import subprocess

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BIN = os.path.join(REPO, "torchlite-cpp_b200", "lib", "tl_token_tests")


def _run(*args):
    assert os.path.exists(BIN), "run python torchlite-cpp_b200/build.py"
    r = subprocess.run([BIN, *args], capture_output=True, text=True, timeout=600)
    return r.returncode, r.stdout + r.stderr


def test_exceptions():
    rc, out = _run("--cpu")
    assert rc == 0, out
    assert "errors ok" in out


@pytest.mark.gpu
def test_on_gpu():
    rc, out = _run()
    assert rc == 0, out
    assert "all token tests passed" in out
