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

import torch

from . import _lib

_E4M3 = torch.float8_e4m3fn
_FLOATS = (torch.bfloat16, torch.float32)


def _fail(what, status):
    if status:
        msg = _lib.load().laya_b200_last_error(None)
        raise RuntimeError(f"{what}: {msg.decode() if msg else 'unknown error'}")


def _rows(name, t, dtypes, columns=None):
    """Check a [..., columns] tensor whose rows lie at one stride; returns
    (rows, columns, row stride)."""
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes:
        raise ValueError(f"{name} must be a tensor of {' or '.join(str(d) for d in dtypes)}")
    if t.dim() < 1 or (columns is not None and t.shape[-1] != columns):
        raise ValueError(f"{name} must have {columns} columns; got shape {tuple(t.shape)}")
    n = t.shape[-1]
    if t.dim() == 2:
        rows, stride = t.shape[0], t.stride(0)
    elif t.dim() == 1:
        rows, stride = 1, n
    else:
        rows = t.numel() // n if n else 0
        stride = t.stride(-2)
        for d in range(t.dim() - 2):
            if t.shape[d] > 1 and t.stride(d) != t.stride(d + 1) * t.shape[d + 1]:
                raise ValueError(f"{name}'s rows must lie at one stride; got strides {t.stride()}")
    if n > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}'s columns must be contiguous")
    return rows, n, (stride if rows > 1 else max(n, 1))


def _contiguous(name, t, shape, dtype):
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or tuple(t.shape) != tuple(shape) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)}")


def _check(device, *tensors):
    if device.type != "cuda":
        raise ValueError("the operators run on CUDA tensors only")
    for t in tensors:
        if t is not None and t.device != device:
            raise ValueError(f"tensors on {t.device} and {device}")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError("the operators record no gradient; call them under torch.no_grad() or on detached tensors")


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
    return None if t is None else t.data_ptr()


class _On:
    """The tensors' device current for the call, and its current stream."""
    __slots__ = ("device", "guard")

    def __init__(self, device):
        self.device = device
        self.guard = None if device.index == torch.cuda.current_device() else torch.cuda.device(device)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        return torch.cuda.current_stream(self.device).cuda_stream

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _rms(x, weight, eps, residual, y, codes, scale):
    rows, d, ldx = _rows("x", x, _FLOATS)
    if not 1 <= d <= 16384:
        raise ValueError("x must have 1 to 16384 columns")
    if not 0 < eps < float("inf"):
        raise ValueError("eps must be positive and finite")
    if weight is not None:
        _contiguous("weight", weight, (d,), torch.float32)
    ldr = 0
    if residual is not None:
        if not isinstance(residual, torch.Tensor) or residual.shape != x.shape:
            raise ValueError(f"residual must have x's shape {tuple(x.shape)}")
        _, _, ldr = _rows("residual", residual, _FLOATS, d)
        if rows > 1 and ldr < d:
            raise ValueError("residual's rows overlap")
        _disjoint("residual", residual, x, weight)
    _check(x.device, x, weight, residual, y)
    ldy = 0
    if y is not None:
        _, _, ldy = _rows("out", y, _FLOATS, d)
        if rows > 1 and ldy < d:
            raise ValueError("out's rows overlap")
        _disjoint("out", y, weight, residual)
        if y.data_ptr() != x.data_ptr() or y.dtype != x.dtype or ldy != ldx:  # in place is allowed
            _disjoint("out", y, x)
    if rows > 1 and ldx < d:
        raise ValueError("x's rows overlap")
    if rows == 0:
        return
    args = _lib.RmsNormArgs(rows, d, eps, x.dtype == torch.float32,
                            residual is not None and residual.dtype == torch.float32,
                            y is not None and y.dtype == torch.float32, x.data_ptr(), ldx, _ptr(residual), ldr,
                            _ptr(weight), _ptr(y), ldy, _ptr(codes), d, _ptr(scale))
    with _On(x.device) as stream:
        _fail("rms_norm", _lib.load().laya_b200_rms_norm(ctypes.byref(args), stream))


def rms_norm(x, weight=None, eps=1e-5, *, residual=None, out=None, dtype=None):
    """y = h * rsqrt(mean(h^2) + eps) * weight over the last axis, h = x + residual.

    ``x``: bf16 or fp32 ``[..., d]`` (d up to 16,384), rows at any stride.
    ``residual`` (bf16 or fp32, x's shape) is updated in place to h; the norm
    reads h before that rounding.  ``weight``: fp32 ``[d]`` or None.  Returns
    ``out`` (``x`` itself is allowed), or a new tensor of ``dtype`` (x's)."""
    if not isinstance(x, torch.Tensor):
        raise ValueError("x must be a tensor")
    if out is None:
        out = torch.empty(x.shape, dtype=dtype or x.dtype, device=x.device)
    elif out.shape != x.shape or (dtype is not None and out.dtype != dtype):
        raise ValueError(f"out must have x's shape {tuple(x.shape)}" + (f" and be {dtype}" if dtype else ""))
    _rms(x, weight, eps, residual, out, None, None)
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
    _rms(x, weight, eps, residual, y, codes, scale)
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


def _lora(x, codes, code_scale, weight, weight_scale, lora_a, lora_b, index, scaling, bias, rows_per_index, out):
    rows, k, ldx = _rows("x", x, (torch.bfloat16,))
    n, _, ldw = _rows("weight", weight, (torch.bfloat16 if codes is None else _E4M3,), k)
    if weight.dim() != 2:
        raise ValueError(f"weight must be [out_features, {k}]")
    if not isinstance(lora_a, torch.Tensor) or lora_a.dim() != 3:
        raise ValueError("lora_a must be [slots, rank, in_features]")
    slots, rank = lora_a.shape[:2]
    _contiguous("lora_a", lora_a, (slots, rank, k), torch.bfloat16)
    _contiguous("lora_b", lora_b, (slots, n, rank), torch.bfloat16)
    if slots < 1 or rank % 8 or not 8 <= rank <= 256:
        raise ValueError("the adapters need at least one slot and a rank that is a multiple of 8 up to 256")
    if rows_per_index < 1:
        raise ValueError("rows_per_index must be positive")
    _contiguous("index", index, (-(-rows // rows_per_index),), torch.int32)
    if scaling is not None:
        _contiguous("scaling", scaling, (slots,), torch.float32)
    if bias is not None:
        _contiguous("bias", bias, (n,), torch.bfloat16)
    ldc = 0
    if codes is not None:
        if not isinstance(codes, torch.Tensor) or codes.shape != x.shape:
            raise ValueError(f"codes must have x's shape {tuple(x.shape)}")
        _, _, ldc = _rows("codes", codes, (_E4M3,), k)
        _contiguous("scale", code_scale, x.shape[:-1], torch.float32)
        _contiguous("weight_scale", weight_scale, (n,), torch.float32)
    if k % (8 if codes is None else 16):
        raise ValueError(f"in_features must be a multiple of {8 if codes is None else 16}")
    given = (x, codes, code_scale, weight, weight_scale, lora_a, lora_b, index, scaling, bias)
    _check(x.device, *given, out)
    if out is None:
        out = torch.empty((*x.shape[:-1], n), dtype=torch.bfloat16, device=x.device)
        ldo = n
    else:
        if out.shape != (*x.shape[:-1], n):
            raise ValueError(f"out must have shape {(*x.shape[:-1], n)}")
        _, _, ldo = _rows("out", out, (torch.bfloat16,), n)
        if rows > 1 and ldo < n:
            raise ValueError("out's rows overlap")
        _disjoint("out", out, *given)
    if rows == 0 or n == 0:
        return out
    args = _lib.LoraArgs(rows, k, n, slots, rank, rows_per_index, x.data_ptr(), ldx, _ptr(codes), ldc,
                         _ptr(code_scale), weight.data_ptr(), ldw, _ptr(weight_scale), lora_a.data_ptr(),
                         lora_b.data_ptr(), _ptr(scaling), index.data_ptr(), _ptr(bias), out.data_ptr(), ldo)
    ref = ctypes.byref(args)
    lib = _lib.load()
    with _On(x.device) as stream:
        size = ctypes.c_size_t()
        _fail("lora_linear", lib.laya_b200_lora_workspace(ref, ctypes.byref(size)))
        work = torch.empty(size.value, dtype=torch.uint8, device=x.device)
        _fail("lora_linear", lib.laya_b200_lora_linear(ref, work.data_ptr(), size.value, stream))
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
