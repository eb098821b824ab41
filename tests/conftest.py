"""Shared fixtures.  `-m "not gpu"` runs on CPU only; `-m gpu` needs an MI355X."""
import json
import os
import subprocess
import sys

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "oracle"))
sys.path.insert(0, os.path.join(ROOT, "cuda-cnn-gan-vae_amd"))
sys.path.insert(0, ROOT)

import oracle_api  # noqa: E402  (test infrastructure: the CPU checker)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu)")


# Tests that expect a value which is wrong, with the reason.  They run as they are and have to fail.
WRONG_EXPECTATIONS = {
    "test_gpu_layernorm.py::test_functions[%d-gelu]" % n:
        "takes the function layer's formula for GeLU's slope, which is not the derivative of GeLU (0.399 at 0, where it is 0.5); "
        "test_gpu_layernorm_edges.py holds the gradient against float64 and against differences"
    for n in (60, 1001, 2048, 20000, 40000)}


def pytest_collection_modifyitems(items):
    for item in items:
        reason = WRONG_EXPECTATIONS.get("%s::%s" % (os.path.basename(str(item.fspath)), item.name))
        if reason:
            item.add_marker(pytest.mark.xfail(reason=reason, raises=AssertionError, strict=True))


@pytest.fixture(scope="session")
def oracle():
    if not oracle_api.available("oracle"):
        subprocess.check_call(["make", "-C", os.path.join(ROOT, "oracle")])
    return oracle_api.Oracle("oracle")


@pytest.fixture(scope="session")
def ref():
    """The reference's own CPU headers, compiled in the authoring container (absent elsewhere -> skip)."""
    if not oracle_api.available("ref"):
        pytest.skip("oracle/_ref/libtensor_ref.so not built (needs /root/reference)")
    return oracle_api.Oracle("ref")


@pytest.fixture(scope="session")
def kat():
    return json.load(open(os.path.join(ROOT, "tests", "golden", "ctensortest_kat.json")))


@pytest.fixture(scope="session")
def golden():
    return np.load(os.path.join(ROOT, "tests", "golden", "ref_vectors.npz"))


def rel_err(got, want):
    """max|got-want| / max|want| per tensor -- the parity metric for fp32 results."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    scale = np.max(np.abs(want))
    return float(np.max(np.abs(got - want)) / (scale if scale > 0 else 1.0))
