"""CPU: the switch of the language-model operators, and scratch memory that they do not need."""
import ctypes as C
import os
import re
import subprocess

import pytest

from deepnet_amd import native

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_attention_option():
    assert '"attention_bf16x3"' in open(os.path.join(ROOT, "include", "tensor_hip.h")).read()
    if os.environ.get("DNH_ATTENTION_BF16X3") is None:
        assert native.get_option("attention_bf16x3") == 1
    with native.option("attention_bf16x3", 0):
        assert native.get_option("attention_bf16x3") == 0
    for bad in (-1, 2):
        with pytest.raises(ValueError):
            native.set_option("attention_bf16x3", bad)


def test_few_tokens_ask_for_next_to_no_scratch_memory():
    """The gradient of up to 512 tokens keeps nothing between launches, however wide the rows are."""
    lib, n = native.load(), C.c_size_t()
    for tokens, width in ((1, 1), (512, 1 << 19), (512, 300), (7, 1 << 23)):
        native.check(lib.dnh_embedding_grad_scratch_bytes(tokens, 50000, width, C.byref(n)))
        assert n.value <= 256, (tokens, width, n.value)
    native.check(lib.dnh_embedding_grad_scratch_bytes(513, 50000, 300, C.byref(n)))
    assert n.value > 513 * 8
    native.check(lib.dnh_embedding_grad_scratch_bytes(512, 50000, 1 << 20, C.byref(n)))       # too much for one launch
    assert n.value > 64 * 2 * (1 << 20) * 8


def test_attention_kernels_are_those_that_calls_reach():
    """Two wavefronts take 33 to 64 rows of single precision; in double precision two hold 32, which the kernel for few rows takes."""
    names = subprocess.run(["nm", native.lib_path()], capture_output=True, text=True, check=True).stdout
    kernels = re.findall(r"attention_kernelINS_6Mma(F32|F64)ELi(\d+)ELi([24])E", names)
    assert {(t, w) for t, _, w in kernels} == {("F32", "2"), ("F32", "4"), ("F64", "4")}
