"""Refusals of the row operators, on the host: what the C entry points and the
Python calls answer to arguments they cannot take, before any CUDA call."""
import ctypes

import pytest
import torch

from laya_b200 import _lib, ops

BASE = 1 << 20


def rms_args(**kw):
    a = dict(rows=4, columns=64, eps=1e-5, x=BASE, x_stride=64, y=BASE, y_stride=64)
    return _lib.RmsNormArgs(**{**a, **kw})


def lora_args(**kw):
    a = dict(rows=4, in_features=64, out_features=64, slots=2, rank=16, rows_per_index=1, x=BASE, x_stride=64,
             weight=BASE, weight_stride=64, lora_a=BASE, lora_b=BASE, index=BASE, out=BASE, out_stride=64)
    return _lib.LoraArgs(**{**a, **kw})


@pytest.mark.parametrize("change, word", [
    (dict(rows=-1), b"rows"), (dict(rows=(1 << 22) + 1), b"rows"), (dict(columns=0), b"columns"),
    (dict(columns=16385), b"columns"), (dict(eps=0.0), b"eps"), (dict(eps=float("nan")), b"eps"),
    (dict(eps=float("inf")), b"eps"), (dict(x=None), b"null"), (dict(y=None), b"neither"),
    (dict(codes=BASE, codes_stride=64), b"together"), (dict(scale=BASE), b"together"),
    (dict(x_stride=63), b"stride"), (dict(y_stride=8), b"stride"), (dict(residual=BASE), b"stride"),
    (dict(x=BASE + 1), b"aligned"), (dict(weight=BASE + 2), b"aligned"),
])
def test_rms_norm_refuses(change, word):
    lib = _lib.load()
    assert lib.laya_b200_rms_norm(ctypes.byref(rms_args(**change)), None) != 0
    assert word in lib.laya_b200_last_error(None)


@pytest.mark.parametrize("change, word", [
    (dict(rows=-1), b"rows"), (dict(rows=(1 << 22) + 1), b"rows"), (dict(in_features=60), b"in_features"),
    (dict(in_features=0), b"in_features"), (dict(out_features=0), b"out_features"), (dict(slots=0), b"slots"),
    (dict(rank=0), b"rank"), (dict(rank=12), b"rank"), (dict(rank=264), b"rank"),
    (dict(rows_per_index=0), b"rows_per_index"), (dict(x=None), b"null"), (dict(index=None), b"null"),
    (dict(codes=BASE, codes_stride=64), b"code_scale"), (dict(x_stride=56), b"stride"),
    (dict(out_stride=63), b"stride"), (dict(x_stride=68), b"16-byte"), (dict(x=BASE + 8), b"16-byte"),
    (dict(weight_stride=65), b"16-byte"), (dict(weight=BASE + 4), b"16-byte"), (dict(lora_a=BASE + 2), b"16-byte"),
    (dict(lora_b=BASE + 8), b"16-byte"), (dict(out=BASE + 1), b"aligned"), (dict(index=BASE + 2), b"aligned"),
    (dict(codes=BASE, codes_stride=72, code_scale=BASE, weight_scale=BASE), b"codes rows"),
    (dict(codes=BASE, codes_stride=72, in_features=72, x_stride=72, weight_stride=72), b"in_features"),
])
def test_lora_linear_refuses(change, word):
    lib = _lib.load()
    assert lib.laya_b200_lora_linear(ctypes.byref(lora_args(**change)), BASE, 1 << 30, None) != 0
    assert word in lib.laya_b200_last_error(None)


def test_null_arguments_and_no_rows():
    lib = _lib.load()
    assert lib.laya_b200_rms_norm(None, None) != 0
    assert lib.laya_b200_lora_linear(None, None, 0, None) != 0
    assert lib.laya_b200_lora_workspace(ctypes.byref(lora_args()), None) != 0
    assert lib.laya_b200_op_status(None) != 0
    # nothing to do is no error, with or without a GPU
    assert lib.laya_b200_rms_norm(ctypes.byref(rms_args(rows=0)), None) == 0
    assert lib.laya_b200_lora_linear(ctypes.byref(lora_args(rows=0)), None, 0, None) == 0


def bf(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def lora_call(**kw):
    a = dict(x=bf(4, 64), weight=bf(32, 64), lora_a=bf(2, 16, 64), lora_b=bf(2, 32, 16),
             index=torch.zeros(4, dtype=torch.int32))
    a.update(kw)
    extra = {k: a[k] for k in a if k not in ("x", "weight", "lora_a", "lora_b", "index")}
    return ops.lora_linear(a["x"], a["weight"], a["lora_a"], a["lora_b"], a["index"], **extra)


@pytest.mark.parametrize("kw", [
    dict(x=bf(4, 64).float()), dict(x=bf(4, 60), weight=bf(32, 60), lora_a=bf(2, 16, 60)), dict(x=bf(64, 4).t()),
    dict(weight=bf(32, 72)), dict(weight=bf(64)), dict(lora_a=bf(2, 12, 64), lora_b=bf(2, 32, 12)),
    dict(lora_a=bf(2, 16, 72)), dict(lora_b=bf(2, 31, 16)), dict(lora_a=bf(0, 16, 64), lora_b=bf(0, 32, 16)),
    dict(index=torch.zeros(4, dtype=torch.int64)), dict(index=torch.zeros(3, dtype=torch.int32)),
    dict(rows_per_index=0), dict(rows_per_index=2), dict(scaling=torch.ones(3)), dict(bias=bf(31)),
    dict(lora_b=bf(2, 16, 32).transpose(1, 2)), dict(),
])
def test_lora_linear_call_refuses(kw):
    with pytest.raises(ValueError):  # the last one: CPU tensors
        lora_call(**kw)


@pytest.mark.parametrize("kw", [
    dict(x=bf(4, 64).half()), dict(x=bf(64, 4).t()), dict(x=bf(4, 0)), dict(x=bf(4, 16385)), dict(eps=0.0),
    dict(eps=float("nan")), dict(weight=torch.ones(63)), dict(weight=bf(64)), dict(residual=bf(4, 63)),
    dict(residual=bf(4, 64).half()), dict(x=torch.zeros(2, 3, 64)[:, ::2].transpose(0, 1)), dict(x="rows"), dict(),
])
def test_rms_norm_call_refuses(kw):
    kw = dict(kw)
    x = kw.pop("x", bf(4, 64))
    for fn in (ops.rms_norm, ops.rms_norm_quant):
        with pytest.raises(ValueError):
            fn(x, kw.get("weight"), kw.get("eps", 1e-5), residual=kw.get("residual"))


def test_stack_adapters():
    a, b, s = ops.stack_adapters([(torch.ones(3, 16), torch.ones(8, 3), 0.5), None,
                                  (torch.ones(10, 16), torch.ones(8, 10), 2.0)], device="cpu")
    assert a.shape == (3, 16, 16) and b.shape == (3, 8, 16) and s.tolist() == [0.5, 0.0, 2.0]
    assert a[0, 3:].abs().sum() == 0 and b[0, :, 3:].abs().sum() == 0 and a[1].abs().sum() == 0
    assert a[2].sum() == 160 and b[2].sum() == 80
    bad = torch.ones(3, 16)
    bad[1, 2] = float("inf")
    for given in ([], [None], [(bad, torch.ones(8, 3), 1.0)], [(torch.ones(3, 16), torch.ones(8, 3), float("nan"))],
                  [(torch.ones(3, 16), torch.ones(8, 4), 1.0)], [(torch.ones(300, 16), torch.ones(8, 300), 1.0)]):
        with pytest.raises(ValueError):
            ops.stack_adapters(given, device="cpu")
    with pytest.raises(ValueError):
        ops.stack_adapters([(torch.ones(10, 16), torch.ones(8, 10), 1.0)], rank=8, device="cpu")

