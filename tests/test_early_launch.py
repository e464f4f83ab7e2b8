"""Kernels that are set up while the one before them still writes (launch_after in rows.cuh).

What such a kernel reads may change while it lives, so a parameter that is promised not to (const
__restrict__: read-only loads, which may be moved above the wait) would be a false promise."""
import glob
import os
import re

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def kernels():
    """name -> (parameters, body) of every __global__ function."""
    found = {}
    for path in glob.glob(os.path.join(REPO, "torchlite-cpp_b200", "csrc", "*.cu")):
        with open(path) as f:
            text = f.read()
        for m in re.finditer(r"__global__[^;{]*?(\w+)\(([^()]*)\)\s*\{", text):
            end = text.index("\n}", m.end())
            found[m.group(1)] = (m.group(2), text[m.end():end])
    return found


def test_what_is_launched_early_waits_and_promises_nothing():
    found = kernels()
    early = set()
    for path in glob.glob(os.path.join(REPO, "torchlite-cpp_b200", "csrc", "*.cu")):
        with open(path) as f:
            early |= set(re.findall(r"launch_after\(\s*(\w+)", f.read()))
    assert {"ln_bwd_finish_kernel", "embed_sum_kernel", "embed_join_kernel"} <= early <= set(found)
    for name in early:
        params, body = found[name]
        assert "after_previous()" in body, name
        assert "__restrict__" not in params, name
