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
operator cannot take raise ValueError before anything is launched.  Inference
only: no operator records a gradient, and tensors that require one are refused
while gradients are enabled.  There is no CPU path.
"""
import ctypes
import functools
import struct

import torch

from . import _lib

_E4M3 = torch.float8_e4m3fn
_BF16, _F32 = torch.bfloat16, torch.float32
_FLOATS = (_BF16, _F32)

# The argument blocks of include/laya_b200.h, packed in C layout: a call's host
# time is what bounds a single row, and this takes a third of what filling a
# ctypes structure does.
_RMS_ARGS = struct.Struct("@2if3i PqPqPPqPqP")
_LORA_ARGS = struct.Struct("@6i PqPqPPqPPPPPPPq")


def _fail(what, status):
    if status:
        msg = _lib.load().laya_b200_last_error(None)
        raise RuntimeError(f"{what}: {msg.decode() if msg else 'unknown error'}")


def _rows(name, t, dtypes, columns=None):
    """Check a [..., columns] tensor whose rows lie at one stride; returns
    (rows, columns, row stride)."""
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes:
        raise ValueError(f"{name} must be a tensor of {' or '.join(str(d) for d in dtypes)}")
    shape, strides = t.shape, t.stride()
    if not shape or (columns is not None and shape[-1] != columns):
        raise ValueError(f"{name} must have {columns or 'some'} columns; got shape {tuple(shape)}")
    n = shape[-1]
    if len(shape) == 2:
        rows, stride = shape[0], strides[0]
    elif len(shape) == 1:
        rows, stride = 1, n
    else:
        rows = t.numel() // n if n else 0
        stride = strides[-2]
        axes = [(m, st) for m, st in zip(shape[:-1], strides[:-1]) if m > 1]
        if axes:
            stride = axes[-1][1]
        for (_, outer), (m, inner) in zip(axes, axes[1:]):
            if outer != inner * m:
                raise ValueError(f"{name}'s rows must lie at one stride; got strides {strides}")
    if n > 1 and strides[-1] != 1:
        raise ValueError(f"{name}'s columns must be contiguous")
    if rows <= 1:
        stride = n
    elif stride < n:
        raise ValueError(f"{name}'s rows overlap")
    return rows, n, stride


def _contiguous(name, t, shape, dtype):
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)}")


def _device(first, *others):
    """Index of the CUDA device that all the tensors are on."""
    index = first.get_device()
    if index < 0:
        raise ValueError("the operators run on CUDA tensors only")
    grad = first.requires_grad
    for t in others:
        if t is not None:
            if t.get_device() != index:
                raise ValueError(f"tensors on {t.device} and {first.device}")
            grad = grad or t.requires_grad
    if grad and torch.is_grad_enabled():
        raise ValueError("the operators record no gradient; call them under torch.no_grad() or on detached tensors")
    return index


def _span(t):
    """[first, last) byte address of what t covers (strides are not negative)."""
    if t.numel() == 0:
        return 0, 0
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _disjoint(name, out, *others):
    lo, hi = _span(out)
    for t in others:
        if t is not None:
            a, b = _span(t)
            if a < hi and lo < b:
                raise ValueError(f"{name} overlaps another argument")


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _launch(what, index, call):
    """call(stream) with device `index` current."""
    if torch.cuda.current_device() == index:
        _fail(what, call(torch._C._cuda_getCurrentRawStream(index)))
    else:
        with torch.cuda.device(index):
            _fail(what, call(torch._C._cuda_getCurrentRawStream(index)))


def _rms(x, weight, eps, residual, y, codes, scale, given):
    """`given`: y is the caller's (it may overlap an argument)."""
    rows, d, ldx = _rows("x", x, _FLOATS)
    if not 1 <= d <= 16384:
        raise ValueError("x must have 1 to 16384 columns")
    if not 0 < eps < float("inf"):
        raise ValueError("eps must be positive and finite")
    if weight is not None:
        _contiguous("weight", weight, (d,), _F32)
    ldr = ldy = 0
    if residual is not None:
        _, _, ldr = _rows("residual", residual, _FLOATS, d)
        if residual.shape != x.shape:
            raise ValueError(f"residual must have x's shape {tuple(x.shape)}")
        _disjoint("residual", residual, x, weight)
    if y is not None:
        ldy = d
        if given:
            _, _, ldy = _rows("out", y, _FLOATS, d)
            _disjoint("out", y, weight, residual)
            if y.data_ptr() != x.data_ptr() or y.dtype != x.dtype or ldy != ldx:  # in place is allowed
                _disjoint("out", y, x)
    index = _device(x, weight, residual, y)
    if rows == 0:
        return
    args = _RMS_ARGS.pack(rows, d, eps, x.dtype is _F32, residual is not None and residual.dtype is _F32,
                          y is not None and y.dtype is _F32, x.data_ptr(), ldx, _ptr(residual), ldr, _ptr(weight),
                          _ptr(y), ldy, _ptr(codes), d, _ptr(scale))
    _launch("rms_norm", index, lambda stream: _lib.load().laya_b200_rms_norm(args, stream))


def rms_norm(x, weight=None, eps=1e-5, *, residual=None, out=None, dtype=None):
    """y = h * rsqrt(mean(h^2) + eps) * weight over the last axis, h = x + residual.

    ``x``: bf16 or fp32 ``[..., d]`` (d up to 16,384), rows at any stride.
    ``residual`` (bf16 or fp32, x's shape) is updated in place to h; the norm
    reads h before that rounding.  ``weight``: fp32 ``[d]`` or None.  Returns
    ``out`` (``x`` itself is allowed), or a new tensor of ``dtype`` (x's)."""
    if not isinstance(x, torch.Tensor):
        raise ValueError("x must be a tensor")
    given = out is not None
    if not given:
        out = torch.empty(x.shape, dtype=dtype or x.dtype, device=x.device)
    elif out.shape != x.shape or (dtype is not None and out.dtype != dtype):
        raise ValueError(f"out must have x's shape {tuple(x.shape)}" + (f" and be {dtype}" if dtype else ""))
    _rms(x, weight, eps, residual, out, None, None, given)
    return out


def rms_norm_quant(x, weight=None, eps=1e-5, *, residual=None, rows=False):
    """``rms_norm`` whose rows come as e4m3 codes and fp32 scales: y ~ codes *
    scale[:, None], scale = max|y| / 448 (at least 1e-12).

    Returns ``(codes, scale)``, with ``rows`` also y in x's type (what the
    adapters of ``lora_linear_fp8`` read)."""
    if not isinstance(x, torch.Tensor) or x.dim() < 1:
        raise ValueError("x must be a tensor of rows")
    codes = torch.empty(x.shape, dtype=_E4M3, device=x.device)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device) if rows else None
    _rms(x, weight, eps, residual, y, codes, scale, False)
    return (codes, scale, y) if rows else (codes, scale)


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


# Workspace bytes by sizes and device (the plan depends on the GPU's SM count).
_workspace = functools.lru_cache(maxsize=4096)(lambda index, *sizes: _query_workspace(*sizes))


def _query_workspace(rows, k, n, slots, rank, per, fp8):
    # any non-null address selects the FP8 plan; nothing is read
    args = _LORA_ARGS.pack(rows, k, n, slots, rank, per, 0, 0, 256 if fp8 else 0, *[0] * 12)
    size = ctypes.c_size_t()
    _fail("lora_linear", _lib.load().laya_b200_lora_workspace(args, ctypes.byref(size)))
    return size.value


def _lora(x, codes, code_scale, weight, weight_scale, lora_a, lora_b, index, scaling, bias, rows_per_index, out):
    fp8 = codes is not None
    rows, k, ldx = _rows("x", x, (_BF16,))
    n, _, ldw = _rows("weight", weight, (_E4M3 if fp8 else _BF16,), k)
    if weight.dim() != 2:
        raise ValueError(f"weight must be [out_features, {k}]")
    if not isinstance(lora_a, torch.Tensor) or lora_a.dim() != 3:
        raise ValueError("lora_a must be [slots, rank, in_features]")
    slots, rank, _ = lora_a.shape
    _contiguous("lora_a", lora_a, (slots, rank, k), _BF16)
    _contiguous("lora_b", lora_b, (slots, n, rank), _BF16)
    if slots < 1 or rank % 8 or not 8 <= rank <= 256:
        raise ValueError("the adapters need at least one slot and a rank that is a multiple of 8 up to 256")
    if rows_per_index < 1:
        raise ValueError("rows_per_index must be positive")
    _contiguous("index", index, (-(-rows // rows_per_index),), torch.int32)
    if scaling is not None:
        _contiguous("scaling", scaling, (slots,), _F32)
    if bias is not None:
        _contiguous("bias", bias, (n,), _BF16)
    ldc = 0
    if fp8:
        _, _, ldc = _rows("codes", codes, (_E4M3,), k)
        if codes.shape != x.shape:
            raise ValueError(f"codes must have x's shape {tuple(x.shape)}")
        _contiguous("scale", code_scale, x.shape[:-1], _F32)
        _contiguous("weight_scale", weight_scale, (n,), _F32)
    if k % (16 if fp8 else 8):
        raise ValueError(f"in_features must be a multiple of {16 if fp8 else 8}")
    device = _device(x, codes, code_scale, weight, weight_scale, lora_a, lora_b, index, scaling, bias, out)
    if out is None:
        out = x.new_empty((*x.shape[:-1], n))
        ldo = n
    else:
        if out.shape != (*x.shape[:-1], n):
            raise ValueError(f"out must have shape {(*x.shape[:-1], n)}")
        _, _, ldo = _rows("out", out, (_BF16,), n)
        _disjoint("out", out, x, codes, code_scale, weight, weight_scale, lora_a, lora_b, index, scaling, bias)
    if rows == 0 or n == 0:
        return out
    args = _LORA_ARGS.pack(rows, k, n, slots, rank, rows_per_index, x.data_ptr(), ldx, _ptr(codes), ldc,
                           _ptr(code_scale), weight.data_ptr(), ldw, _ptr(weight_scale), lora_a.data_ptr(),
                           lora_b.data_ptr(), _ptr(scaling), index.data_ptr(), _ptr(bias), out.data_ptr(), ldo)

    def call(stream):
        # the caching allocator hands this memory to later work of this stream only
        size = _workspace(device, rows, k, n, slots, rank, rows_per_index, fp8)
        work = torch.empty(size, dtype=torch.uint8, device=x.device)
        return _lib.load().laya_b200_lora_linear(args, work.data_ptr(), size, stream)

    _launch("lora_linear", device, call)
    return out


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
    return _lora(x, None, None, weight, None, lora_a, lora_b, index, scaling, bias, rows_per_index, out)


def lora_linear_fp8(codes, scale, weight, weight_scale, x, lora_a, lora_b, index, *, scaling=None, bias=None,
                    rows_per_index=1, out=None):
    """``lora_linear`` whose shared projection runs on e4m3: ``codes``
    ``[..., k]`` with ``scale`` per row (as ``rms_norm_quant`` writes them; k a
    multiple of 16) times ``weight`` e4m3 ``[n, k]`` with ``weight_scale`` fp32
    ``[n]``.  The adapters read the bf16 rows ``x``."""
    if codes is None:
        raise ValueError("codes must be an e4m3 tensor")
    return _lora(x, codes, scale, weight, weight_scale, lora_a, lora_b, index, scaling, bias, rows_per_index, out)


def op_status(device=None):
    """Nonzero when a bounded wait inside an operator ran out on ``device``
    since the last call (its output is invalid); synchronises the device."""
    with torch.cuda.device(device):
        torch.cuda.synchronize()
        status = ctypes.c_int32()
        _fail("op_status", _lib.load().laya_b200_op_status(ctypes.byref(status)))
    return status.value
