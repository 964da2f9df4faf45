"""The row operators beside autograd: what they write in place counts as changed,
and tangents are refused as gradients are."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from laya_b200 import ops

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF16 = torch.bfloat16


def lora_inputs(m=4):
    g = torch.Generator(device=DEV).manual_seed(1)

    def randn(*shape):
        return torch.randn(shape, generator=g, device=DEV).to(BF16)

    return [randn(m, 64), randn(32, 64), randn(2, 8, 64), randn(2, 32, 8),
            torch.zeros(m, dtype=torch.int32, device=DEV)]


def saved(t):
    """A loss whose backward pass reads t."""
    w = torch.ones_like(t, requires_grad=True)
    return w, (w * t).sum()


def writes():
    x = torch.randn(4, 64, device=DEV)
    wide = torch.randn(4, 200, device=DEV)
    return {"residual": (wide[:, 8:72], lambda t: ops.rms_norm(x, residual=t)),
            "residual, codes": (wide[:, 8:72].clone(), lambda t: ops.rms_norm_quant(x, residual=t)),
            "norm's out": (torch.randn(4, 64, device=DEV), lambda t: ops.rms_norm(x, out=t)),
            "norm in place": (x.clone(), lambda t: ops.rms_norm(t, out=t)),
            "projection's out": (torch.randn(4, 32, device=DEV).to(BF16),
                                 lambda t: ops.lora_linear(*lora_inputs(), out=t))}


@pytest.mark.parametrize("which", ["residual", "residual, codes", "norm's out", "norm in place", "projection's out"])
def test_what_is_written_counts_as_changed(which):
    target, call = writes()[which]
    _, loss = saved(target)
    before = target._version
    call(target)
    assert target._version == before + 1
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()
    # of a view, the whole; and what is only read does not count
    base = torch.randn(4, 400, device=DEV)
    view = base[:, :target.shape[1]]
    if target.dtype == base.dtype:
        _, loss = saved(base)
        call(view)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            loss.backward()


def test_what_is_read_does_not_count():
    x = torch.randn(4, 64, device=DEV)
    args = lora_inputs()
    w, loss = saved(x)
    w2, loss2 = saved(args[0])
    ops.rms_norm(x)
    ops.rms_norm_quant(x, rows=True)
    ops.lora_linear(*args)
    loss.backward()
    loss2.backward()
    assert torch.equal(w.grad, x) and torch.equal(w2.grad, args[0])


def test_inference_tensors_are_written():
    with torch.inference_mode():
        h, x = torch.zeros(4, 64, device=DEV), torch.ones(4, 64, device=DEV)
        y = ops.rms_norm(x, residual=h)
    ops.rms_norm(x, residual=h)
    with torch.inference_mode():
        ops.rms_norm(x, residual=h, out=y)
        ops.lora_linear(*lora_inputs(), out=torch.empty(4, 32, dtype=BF16, device=DEV))
    assert (h == 3).all()


def test_tangents_are_refused():
    x, r = torch.randn(4, 64, device=DEV), torch.randn(4, 64, device=DEV)
    args, before = lora_inputs(), r.clone()
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                with pytest.raises(ValueError, match="tangent"):
                    ops.rms_norm(dual)
                with pytest.raises(ValueError, match="tangent"):
                    ops.rms_norm_quant(x, residual=fwd.make_dual(r, torch.ones_like(r)))
                for i in range(4):
                    given = list(args)
                    given[i] = fwd.make_dual(args[i], torch.ones_like(args[i]))
                    with pytest.raises(ValueError, match="tangent"):
                        ops.lora_linear(*given)
        assert torch.equal(ops.rms_norm(fwd.unpack_dual(dual).primal), ops.rms_norm(x))
    assert torch.equal(r, before) and ops.op_status() == 0
