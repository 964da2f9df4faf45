"""Refusals of the row operators that test_ops_cpu.py does not reach: values at the
ends of their types.  CPU tensors are refused too, so each test names the reason."""
import pytest
import torch

from laya_b200 import ops
from test_ops_cpu import bf, lora_call


@pytest.mark.parametrize("eps", [1e-50, 1e39])
def test_eps_that_fp32_does_not_hold(eps):
    for fn in (ops.rms_norm, ops.rms_norm_quant):
        with pytest.raises(ValueError, match="eps"):
            fn(bf(4, 64), None, eps)
        with pytest.raises(ValueError, match="CUDA"):
            fn(bf(4, 64), None, 1e-30)


@pytest.mark.parametrize("per", [2 ** 31, 2 ** 63 - 2, 2 ** 63 - 1])
def test_one_index_for_all_rows(per):
    with pytest.raises(ValueError, match="CUDA"):  # the index has the right length
        lora_call(index=torch.zeros(1, dtype=torch.int32), rows_per_index=per)
    with pytest.raises(ValueError, match="index"):
        lora_call(index=torch.zeros(2, dtype=torch.int32), rows_per_index=per)
