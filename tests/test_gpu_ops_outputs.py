"""Outputs that are columns of wider rows: nothing beside them is written, whatever
their width, start and stride."""
import pytest
import torch

from laya_b200 import ops
from test_gpu_ops import BF16, DEV, call, check_lora, make, runs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m, k, base", [(6, 128, 130), (64, 128, 300), (300, 128, 2000), (2000, 64, 640), (9000, 64, 40)])
@pytest.mark.parametrize("fp8", [False, True])
def test_projection_beside_other_columns(m, k, base, fp8):
    """Rows on 16-byte boundaries and off them, widths that end inside 16 bytes."""
    for n in range(base, base + 9):
        s = make(m + n, m, k, n, 16, 5, fp8, bias=n % 2 == 0)
        index = runs(n, m, min(m, 20), 5)
        ref = check_lora(s, index)
        for lo in (0, 8, 3):
            for behind in ((-n - lo) % 8, (-n - lo) % 8 + 8, 1):  # strides that are multiples of 8, and one behind
                whole = torch.full((m + 1, lo + n + behind), 7.0, dtype=BF16, device=DEV)
                call(s, index, out=whole[:m, lo:lo + n])
                assert torch.equal(whole[:m, lo:lo + n], ref)
                assert (whole[:, :lo] == 7).all() and (whole[:, lo + n:] == 7).all() and (whole[m] == 7).all()
    assert ops.op_status() == 0
