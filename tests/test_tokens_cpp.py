"""The C++ class qmlp::Tokens used from C++: tests/cpp/test_tokens_api.cpp, linked against libqmlp.so. The host part runs everywhere; the device part
takes a layer of experts and its gradients through numbers whose results are exact."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CPP_DIR = os.path.join(ROOT, "tests", "cpp")
BINARY = os.path.join(CPP_DIR, "test_tokens_api")


def run(*args):
    env = dict(os.environ, QMLP_CACHE_DIR=os.path.join(ROOT, "quick-mlp_amd", ".kernel_cache"))
    r = subprocess.run([BINARY, *args], env=env, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "all checks passed" in r.stdout, r.stdout + r.stderr


def test_host_part():
    subprocess.run(["make", "-C", CPP_DIR, "test_tokens_api"], check=True, capture_output=True)
    run("--host")


@pytest.mark.gpu
def test_device_part():
    if os.environ.get("QMLP_WARM_CACHE"):
        pytest.skip("kernels are compiled by qmlp.tokens.precompile")
    assert os.path.exists(BINARY), "tests/cpp/test_tokens_api is missing: run __graft_entry__.build() first"
    run()
