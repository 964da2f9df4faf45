"""Adapter pools past 2^31 elements: the slots at both ends and around the border,
the others holding NaN."""
import pytest
import torch

from test_gpu_ops import BF16, DEV, call, lora_reference, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m, k, n, rank", [(6, 2048, 2048, 16),      # single dot products
                                           (64, 2048, 2048, 256),  # tiles of few rows
                                           (700, 2048, 2048, 16)])   # tiles of many
@pytest.mark.parametrize("fp8", [False, True])
def test_far_slots(m, k, n, rank, fp8):
    s = make(m + rank, m, k, n, rank, 5, fp8)
    slots = (1 << 31) // (rank * k) + 3
    far = [0, 1, slots - 4, slots - 3, slots - 1]  # slot slots - 3 begins at element 2^31
    pools = {}
    for key, shape in (("a", (slots, rank, k)), ("b", (slots, n, rank))):
        pools[key] = torch.full(shape, float("nan"), dtype=BF16, device=DEV)
        pools[key][far] = s[key]
    scaling = torch.full((slots,), float("nan"), device=DEV)
    scaling[far] = s["scaling"]
    own = torch.arange(m, device=DEV) // 3 % 6 - 1
    index = torch.where(own < 0, -1, torch.tensor(far, device=DEV)[own.clamp_min(0)]).to(torch.int32)
    y, tol = lora_reference(s, own)
    out = call(dict(s, a=pools["a"], b=pools["b"], scaling=scaling), index)
    assert ((out.double() - y).abs() <= tol).all()
