"""CPU: the switch of the language-model operators."""
import os

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
