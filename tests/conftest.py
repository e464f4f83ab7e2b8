import os
import sys

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(REPO, "torchlite-cpp_b200")
for p in (REPO, PKG, os.path.dirname(os.path.abspath(__file__))):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA (B200) device")


def pytest_collection_modifyitems(items):
    """Without the reference library's build (oracle/_ref) the benchmark line's test cannot pass: it comes
    last then, so that a run that stops at the first failure has run all others."""
    if not os.path.exists(os.path.join(REPO, "oracle", "_ref")):
        items.sort(key=lambda item: item.name == "test_our_arm_line")


@pytest.fixture(scope="session")
def golden():
    import numpy as np
    path = os.path.join(REPO, "tests", "golden", "reference_matmul.npz")
    with np.load(path) as z:
        return {k: z[k] for k in z.files}


@pytest.fixture(scope="session")
def golden_meta():
    import json
    with open(os.path.join(REPO, "tests", "golden", "reference_matmul.json")) as f:
        return json.load(f)
