"""The entry points between csrc/torch/nodes.cpp and the kernels have one
declaration, which both sides include (no GPU)."""

import os
import re
import subprocess

import pytest

from conftest import ROOT

API = os.path.join(ROOT, "csrc", "hip", "nodes_api.h")
USERS = [os.path.join(ROOT, "csrc", *p) for p in (
    ("hip", "dense.hip"), ("hip", "distill.hip"), ("hip", "toplogits.hip"), ("torch", "nodes.cpp"))]


def compiles(body, tmp_path):
    src = tmp_path / "t.cpp"
    src.write_text('#include "{}"\n{}\n'.format(API, body))
    r = subprocess.run(["g++", "-fsyntax-only", "-std=c++17", "-D__HIP_PLATFORM_AMD__",
                        "-I/opt/rocm/include", str(src)], capture_output=True, text=True)
    return r.returncode == 0, r.stderr


@pytest.mark.skipif(not os.path.exists("/opt/rocm/include/hip/hip_runtime_api.h"),
                    reason="no HIP headers")
def test_a_changed_argument_does_not_compile(tmp_path):
    ok, err = compiles('extern "C" int64_t cer_top_ws(int, int, int, int, int) { return 0; }',
                       tmp_path)
    assert ok, err
    for changed in ("int64_t cer_top_ws(int, int, int, int, int64_t) { return 0; }",
                    "int64_t cer_dense_ws(int, int, int, int, int, int) { return 0; }"):
        assert not compiles('extern "C" ' + changed, tmp_path)[0], changed


def test_both_sides_include_it_and_declare_nothing_else():
    with open(API) as f:
        names = set(re.findall(r"\bcer_\w+", f.read().split('extern "C"')[1]))
    assert len(names) == 13
    for path in USERS:
        with open(path) as f:
            text = f.read()
        assert re.search(r'#include "(\.\./hip/)?nodes_api\.h"', text), path
        # every name that crosses is in the header; prototypes are nowhere else
        if path.endswith("nodes.cpp"):
            assert set(re.findall(r"\bcer_[a-z0-9_]+(?=[(\s])", text)) <= names
            assert 'extern "C"' not in text
        else:
            defined = set(re.findall(r"CER_API (?:int|int64_t) (cer_\w+)\(", text))
            assert defined <= names, defined - names
