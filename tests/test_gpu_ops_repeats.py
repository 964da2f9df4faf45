"""Repeated calls give the same bits: no sum's order depends on which CTA is first."""
import pytest
import torch

from laya_b200 import ops
from test_gpu_ops import BF16, DEV, call, gen, make, randn, runs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m, k, n, rank, slots", [
    (1, 1024, 1024, 16, 1), (64, 1024, 5248, 16, 64), (64, 8192, 72, 200, 37),  # rows by themselves, split K
    (1536, 2624, 1024, 32, 8), (777, 1008, 1543, 24, 5),                        # few tiles of a long K, odd sizes
    (8192, 1024, 5248, 64, 32), (6500, 2624, 1024, 16, 16)])                    # a tile for every pair, several
@pytest.mark.parametrize("fp8", [False, True])
def test_projection(m, k, n, rank, slots, fp8):
    s = make(m + n, m, k, n, rank, slots, fp8, bias=True)
    other = make(m + n + 1, m, k, n, rank, slots, fp8)
    index, shifted = runs(m, m, min(m, 64), slots), runs(m + 1, m, min(m, 9), slots)
    first = call(s, index)
    for i in range(40):
        if i % 3 == 0:
            call(other, shifted)
        assert torch.equal(call(s, index), first)
    assert ops.op_status() == 0


@pytest.mark.parametrize("rows, d", [(1, 1024), (1237, 2623), (32768, 1024), (3000, 8192)])
def test_norm(rows, d):
    x, h = randn(gen(d), rows, d, dtype=BF16), randn(gen(rows), rows, d)
    w = torch.rand(d, device=DEV)
    first = None
    for _ in range(20):
        r = h.clone()
        codes, scale, y = ops.rms_norm_quant(x, w, residual=r, rows=True)
        got = (codes.view(torch.uint8), scale, y, r)
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))
