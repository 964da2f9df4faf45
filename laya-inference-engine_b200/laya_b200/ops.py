"""Row operators of liblaya_b200.so on torch tensors, for blocks that a host
runs beside the engine (no counterpart in the reference):

* ``rms_norm`` / ``rms_norm_quant``: residual addition, RMS norm, and e4m3
  codes with a scale per row (the engine's activation recipe);
* ``lora_linear`` / ``lora_linear_fp8``: a projection with the low-rank
  adapters of many requests beside the shared weight, on bf16 rows or on the
  codes that ``rms_norm_quant`` writes; ``stack_adapters`` lays adapters of
  different rank out for them.

A block runs them one after the other: the norm's codes are the operand of
the FP8 projection, its bf16 rows what the adapters read, and the projection's
output the next norm's ``x``.  Every call runs on its tensors' device and that
device's current stream, does not synchronise, allocates through torch's
allocator only, and can be captured into a CUDA graph.  Arguments that an
operator cannot take raise ValueError before anything is launched (sizes past the
library's limits and operand rows off the 16-byte boundaries: RuntimeError, with
its message).  Inference only: no operator records a gradient or computes a
tangent; tensors that require one are refused while gradients are enabled, and
tensors that carry the other.  What a call writes in place counts as changed for
autograd.  There is no CPU path.
"""
import ctypes
import importlib.util
from pathlib import Path

import torch

from . import _lib


def _load():
    """The native calls (csrc/torch_ops.cpp, built beside the library)."""
    path = Path(__file__).resolve().with_name("_torch_ops.so")
    if not path.exists():
        raise RuntimeError(f"{path.name} is not built; run `python laya-inference-engine_b200/build.py` with torch "
                           "installed (the operators have no other path)")
    spec = importlib.util.spec_from_file_location(f"{__package__}._torch_ops", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


_native = _load()


def rms_norm(x, weight=None, eps=1e-5, *, residual=None, out=None, dtype=None):
    """y = h * rsqrt(mean(h^2) + eps) * weight over the last axis, h = x + residual.

    ``x``: bf16 or fp32 ``[..., d]`` (d up to 16,384), rows at any stride.
    ``residual`` (bf16 or fp32, x's shape) is updated in place to h; the norm
    reads h before that rounding.  ``weight``: fp32 ``[d]`` or None.  Returns
    ``out`` (``x`` itself is allowed), or a new tensor of ``dtype`` (x's).
    ``residual`` and ``out`` may be other columns of x's rows; what shares bytes
    with another argument is refused."""
    return _native.rms_norm(x, weight, eps, residual, out, dtype)


def rms_norm_quant(x, weight=None, eps=1e-5, *, residual=None, rows=False):
    """``rms_norm`` whose rows come as e4m3 codes and fp32 scales: y ~ codes *
    scale[:, None], scale = max|y| / 448 (at least 1e-12).

    Returns ``(codes, scale)``, with ``rows`` also y in x's type (what the
    adapters of ``lora_linear_fp8`` read)."""
    return _native.rms_norm_quant(x, weight, eps, residual, rows)


def stack_adapters(adapters, rank=None, device="cuda"):
    """``(lora_a, lora_b, scaling)`` for ``lora_linear`` from a list of ``(a
    [r, k], b [n, r], scaling)``, one slot each: ranks are padded with zeros to
    ``rank`` (default: the largest, rounded up to a multiple of 8).  None in
    the list leaves its slot zero.  Non-finite adapters are refused."""
    given = [x for x in adapters if x is not None]
    if not given:
        raise ValueError("no adapter")
    k, n = given[0][0].shape[1], given[0][1].shape[0]
    most = max(a.shape[0] for a, _, _ in given)
    rank = (most + 7) // 8 * 8 if rank is None else rank
    if rank % 8 or not 8 <= rank <= 256 or most > rank:
        raise ValueError("rank must be a multiple of 8 up to 256 that no adapter exceeds")
    lora_a = torch.zeros((len(adapters), rank, k), dtype=torch.bfloat16)
    lora_b = torch.zeros((len(adapters), n, rank), dtype=torch.bfloat16)
    scaling = torch.zeros(len(adapters), dtype=torch.float32)
    for i, x in enumerate(adapters):
        if x is None:
            continue
        a, b, s = x
        if a.dim() != 2 or b.dim() != 2 or a.shape[1] != k or b.shape != (n, a.shape[0]):
            raise ValueError(f"adapter {i}: a {tuple(a.shape)} and b {tuple(b.shape)} do not fit [r, {k}] and [{n}, r]")
        lora_a[i, :a.shape[0]] = a
        lora_b[i, :, :a.shape[0]] = b
        scaling[i] = s
        if not (lora_a[i].isfinite().all() and lora_b[i].isfinite().all() and scaling[i].isfinite()):
            raise ValueError(f"adapter {i} contains NaN or infinity")
    return lora_a.to(device), lora_b.to(device), scaling.to(device)


def lora_linear(x, weight, lora_a, lora_b, index, *, scaling=None, bias=None, rows_per_index=1, out=None):
    """x W^T + bias + scaling[a] (x A_a^T) B_a^T, a the adapter of each row.

    ``x``: bf16 ``[..., k]`` (k a multiple of 8, rows on 16-byte boundaries);
    ``weight``: bf16 ``[n, k]``; ``lora_a``: bf16 ``[slots, rank, k]`` and
    ``lora_b``: bf16 ``[slots, n, rank]``, rank a multiple of 8 up to 256 (a
    slot of smaller rank has zeros in the rest); ``scaling``: fp32 ``[slots]``;
    ``bias``: bf16 ``[n]``.  Row m takes adapter ``index[m // rows_per_index]``
    (int32); an index outside ``[0, slots)`` means none.  Sums are fp32 and the
    result is rounded to bf16 once.  The adapters must be finite (rows of
    different slots share matrix instructions)."""
    return _native.lora(x, None, None, weight, None, lora_a, lora_b, index, scaling, bias, rows_per_index, out)


def lora_linear_fp8(codes, scale, weight, weight_scale, x, lora_a, lora_b, index, *, scaling=None, bias=None,
                    rows_per_index=1, out=None):
    """``lora_linear`` whose shared projection runs on e4m3: ``codes``
    ``[..., k]`` with ``scale`` per row (as ``rms_norm_quant`` writes them; k a
    multiple of 16) times ``weight`` e4m3 ``[n, k]`` with ``weight_scale`` fp32
    ``[n]``.  The adapters read the bf16 rows ``x``."""
    if codes is None:
        raise ValueError("codes must be an e4m3 tensor")
    return _native.lora(x, codes, scale, weight, weight_scale, lora_a, lora_b, index, scaling, bias, rows_per_index,
                        out)


def op_status(device=None):
    """Nonzero when a bounded wait inside an operator ran out on ``device``
    since the last call (its output is invalid); synchronises the device, so not
    while any thread captures a graph there."""
    with torch.cuda.device(device):
        torch.cuda.synchronize()
        status, lib = ctypes.c_int32(), _lib.load()
        if lib.laya_b200_op_status(ctypes.byref(status)):
            raise RuntimeError(f"op_status: {(lib.laya_b200_last_error(None) or b'unknown error').decode()}")
    return status.value
