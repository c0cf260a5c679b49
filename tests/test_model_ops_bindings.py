"""The language-model operators in the other host layers: the C++ header through its own driver (tests/cpp/model_ops_test.cpp, built
by __graft_entry__.build()), the F# binding by a static check against the header's declarations."""
import os
import re
import subprocess

import pytest

from deepnet_amd import abi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EXE = os.path.join(ROOT, "tests", "cpp", "_build", "model_ops_test")
NATIVE = open(os.path.join(ROOT, "deepnet_amd", "fsharp", "Hip", "HipNative.fs")).read()
FRONTEND = open(os.path.join(ROOT, "deepnet_amd", "fsharp", "Hip", "HipFrontend.fs")).read()


@pytest.mark.gpu
def test_cpp_model_operators():
    if not os.path.exists(EXE):
        import __graft_entry__
        __graft_entry__.build_cpp_model_test()
    p = subprocess.run([EXE], capture_output=True, text=True, timeout=110)
    assert p.returncode == 0 and " 0 failed" in p.stdout, p.stdout[-2000:] + p.stderr[-2000:]
    assert p.stdout.count("PASS ") >= 18


def test_fsharp_binds_every_operator():
    """Every operator and scratch query has a DllImport, and HipModel passes each as many descriptors as the header's declaration takes
    (the argument kinds of each import are checked with all others)."""
    for name, args in abi.MODEL_OP_SIGNATURES.items():
        assert re.search(rf'EntryPoint="dnh_{name}"\)>\] extern int {name} \(', NATIVE), name
        calls = re.findall(rf"Native\.{name} \(([^)]*)\)", FRONTEND)
        assert calls, f"HipModel does not call {name}"
        for c in calls:
            parts = [x.strip() for x in c.split(",")]
            assert len(parts) == len(args) + 1 and parts[-1] == "Cfg.Stream", (name, parts)
            n = sum(a is abi.OP_SIGNATURES["copy"][0] for a in args)
            assert [x for x in parts if x.startswith("p.[")] == [f"p.[{i}]" for i in range(n)], (name, parts)
    for name in abi.SCRATCH_QUERY_SIGNATURES:
        assert f"extern int dnh_{name} (" in NATIVE


def test_header_documents_every_operator():
    header = open(os.path.join(ROOT, "include", "tensor_hip.h")).read()
    for name in list(abi.MODEL_OP_SIGNATURES) + list(abi.SCRATCH_QUERY_SIGNATURES):
        assert header.count(f"int32_t dnh_{name}(") == 1
