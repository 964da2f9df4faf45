"""The projection's workspace: V, and for many rows the adapters of every 256."""
import ctypes

import pytest
import torch

from laya_b200 import _lib

pytestmark = pytest.mark.gpu


def bytes_of(rows, n, k, rank):
    lib, got = _lib.load(), ctypes.c_size_t()
    args = _lib.LoraArgs(rows=rows, in_features=k, out_features=n, slots=64, rank=rank, rows_per_index=1)
    torch.cuda.init()
    assert lib.laya_b200_lora_workspace(ctypes.byref(args), ctypes.byref(got)) == 0
    return got.value


def up(x):
    return (x + 255) // 256 * 256


@pytest.mark.parametrize("rows, n, k, rank", [(8192, 5248, 1024, 64), (100000, 1024, 2624, 8), (777, 1543, 1000, 24)])
def test_lists_hold_adapters_alone(rows, n, k, rank):
    # 128 bytes of V a row and 32 ranks; a list: a count on a 16-byte boundary, 256 adapters
    assert bytes_of(rows, n, k, rank) == up(rows * ((rank + 31) // 32) * 128) + up((rows + 255) // 256 * 4 * (4 + 256))


@pytest.mark.parametrize("rows, n, k, rank", [(1, 1024, 1024, 16), (64, 5248, 1024, 16), (222, 320, 1504, 40)])
def test_few_rows_take_no_lists(rows, n, k, rank):
    assert bytes_of(rows, n, k, rank) == up(rows * ((rank + 31) // 32) * 128)
