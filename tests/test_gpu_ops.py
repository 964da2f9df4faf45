"""The row operators (laya_b200.ops) against their definitions in 64 bits.

Tolerances, from the arithmetic:

* a result rounded to bf16 is off by at most 2^-8 of itself, one in fp32 by
  2^-24, an e4m3 code by 2^-4 (2^-10 below the smallest normal, 2^-6);
* fp32 sums: a term passes at most ``adds`` additions, each off by 2^-24 of the
  running value (CUDA cores) or 2^-22 (tensor cores, which may cut the aligned
  products off instead of rounding them), so a sum is off by that many steps
  of the sum of the terms' magnitudes.
"""
import pytest
import torch

from laya_b200 import ops

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, std=1.0, dtype=F32):
    return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)


# --------------------------------------------------------------- RMS norm
def rms_reference(x, weight, eps, residual):
    h = x.double()
    if residual is not None:
        h = h + residual.double()
    y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps)
    return h, y if weight is None else y * weight.double()


def y_bound(y, dtype):
    # h 2^-24; its square's sum at most 32 + 5 + 32 additions deep; rsqrt 2
    # steps, two products: under 2 + 40 + 4 steps of 2^-24 (half of the sum's
    # error reaches the root)
    return y.abs() * (64 * 2.0 ** -24 + (2.0 ** -8 if dtype == BF16 else 0)) + 1e-30


def check_rms(x, weight, residual, quant, eps=1e-5, keep=True):
    h_ref, y_ref = rms_reference(x, weight, eps, residual)
    sum_ref = None if residual is None else (x.float() + residual.float()).to(residual.dtype)
    if quant:
        out = ops.rms_norm_quant(x, weight, eps, residual=residual, rows=keep)
        codes, scale = out[0], out[1]
        y = out[2] if keep else None
        assert codes.dtype == torch.float8_e4m3fn and codes.shape == x.shape and scale.shape == x.shape[:-1]
        s_ref = y_ref.abs().amax(-1) / 448
        assert ((scale.double() - s_ref).abs() <= s_ref * 70 * 2.0 ** -24 + 1.01e-12).all()
        q_ref = y_ref / s_ref.clamp_min(1e-12)[..., None]
        # the quotient itself is off by the 2 * 64 + 8 steps of y and scale
        tol = q_ref.abs() * (2.0 ** -4 + 140 * 2.0 ** -24) + 2.0 ** -10
        assert ((codes.double() - q_ref).abs() <= tol).all()
    else:
        y = ops.rms_norm(x, weight, eps, residual=residual)
    if y is not None:
        assert y.dtype == x.dtype
        assert ((y.double() - y_ref).abs() <= y_bound(y_ref, y.dtype)).all()
    if residual is not None:
        assert torch.equal(residual, sum_ref)


@pytest.mark.parametrize("rows, d", [(1, 1), (3, 7), (5, 8), (2, 33), (130, 64), (1, 1000), (9, 1024), (257, 1032),
                                     (31, 2623), (17, 4096), (4, 8191), (6, 16384), (3, 16383)])
@pytest.mark.parametrize("x_type, r_type", [(BF16, F32), (BF16, BF16), (F32, F32), (F32, None), (BF16, None),
                                            (F32, BF16)])
def test_rms_norm(rows, d, x_type, r_type):
    g = gen(rows * 31 + d)
    for quant in (False, True):
        x = randn(g, rows, d, dtype=x_type)
        r = None if r_type is None else randn(g, rows, d, std=3.0, dtype=r_type)
        w = 1 + randn(g, d, std=0.2) if rows % 2 else None
        check_rms(x, w, r, quant, keep=d % 2 == 0)


def test_rms_norm_strides_views_and_types():
    g = gen(5)
    # rows of a wider matrix, on 16-byte boundaries and off them; three axes;
    # one odd start only for one of the buffers
    big = randn(g, 40, 4000, dtype=BF16)
    wide = randn(g, 40, 4000)
    for lo, d in ((0, 1024), (8, 1024), (1, 1024), (3, 1000), (16, 2056)):
        check_rms(big[:, lo:lo + d], None, wide[:, lo:lo + d].clone(), True)
        before = wide.clone()
        r = wide[:, lo:lo + d]
        _, y = rms_reference(big[:, 8:8 + d], None, 1e-5, r)
        got = ops.rms_norm(big[:, 8:8 + d], residual=r)
        assert ((got.double() - y).abs() <= y_bound(y, BF16)).all()
        before[:, lo:lo + d] += big[:, 8:8 + d].float()
        assert torch.equal(wide, before)  # nothing beside the rows was touched
    x3 = randn(g, 5, 6, 128, dtype=BF16)
    check_rms(x3, None, None, True)
    check_rms(randn(g, 128, dtype=BF16), None, None, True)
    # fp32 rows to bf16, into a given buffer, in place
    x = randn(g, 12, 96)
    out = torch.full((12, 200), 7.0, device=DEV, dtype=BF16)
    _, y = rms_reference(x, None, 1e-5, None)
    assert ops.rms_norm(x, out=out[:, 4:100], dtype=BF16).data_ptr() == out[:, 4:100].data_ptr()
    assert ((out[:, 4:100].double() - y).abs() <= y_bound(y, BF16)).all()
    assert (out[:, :4] == 7).all() and (out[:, 100:] == 7).all()
    ops.rms_norm(x, out=x)
    assert ((x.double() - y).abs() <= y_bound(y, F32)).all()
    assert ops.rms_norm(torch.empty(0, 64, device=DEV)).shape == (0, 64)
    codes, scale = ops.rms_norm_quant(torch.empty(0, 64, device=DEV))
    assert codes.shape == (0, 64) and scale.shape == (0,)


def test_rms_norm_rows_without_numbers():
    """Zero rows, infinities and NaN stay in their rows."""
    g = gen(6)
    for d in (64, 1000, 1001, 4096):
        clean = randn(g, 6, d)
        x = clean.clone()
        x[1] = 0
        x[2, d // 2] = float("nan")
        x[3, 5] = float("inf")
        codes, scale, y = ops.rms_norm_quant(x, rows=True)
        c0, s0, y0 = ops.rms_norm_quant(clean, rows=True)
        for i in (0, 4, 5):
            assert torch.equal(codes[i].float(), c0[i].float()) and scale[i] == s0[i] and torch.equal(y[i], y0[i])
        assert (y[1] == 0).all() and (codes[1].float() == 0).all() and scale[1] == torch.tensor(1e-12, device=DEV)
        assert y[2].isnan().all() and codes[2].float().isnan().all() and scale[2].isnan()
        # 1 / sqrt(inf) = 0: the infinity times zero is NaN, the rest zero
        assert y[3, 5].isnan() and (y[3, :5] == 0).all() and codes[3].float().isnan().all() and scale[3].isnan()
        # an infinite weight makes one infinite column: scale inf, the others' codes 0
        w = torch.ones(d, device=DEV)
        w[3] = float("inf")
        codes, scale = ops.rms_norm_quant(clean, w)
        assert scale.isinf().all() and codes[:, 3].float().isnan().all() and (codes[:, 4:].float() == 0).all()


def test_rms_norm_many_rows():
    """More than 2^31 elements: rows at both ends and around the 32-bit border."""
    rows, d = (1 << 19) + 3, 4104
    x = torch.empty(rows, d, dtype=BF16, device=DEV)
    at = [0, 1, (1 << 31) // d, (1 << 31) // d + 1, rows - 1]
    x.fill_(0.25)
    x[at] = randn(gen(8), len(at), d, dtype=BF16)
    y = ops.rms_norm(x)
    _, ref = rms_reference(x[at], None, 1e-5, None)
    assert ((y[at].double() - ref).abs() <= y_bound(ref, BF16)).all()
    assert (y[12345] == 1).all() and (y[rows - 2] == 1).all()


# ---------------------------------------------------------------- adapters
def quantise(x):
    scale = (x.float().abs().amax(-1) / 448).clamp_min(1e-12)
    return (x.float() / scale[..., None]).to(torch.float8_e4m3fn), scale


def make(seed, m, k, n, rank, slots, fp8=False, bias=False):
    g = gen(seed)
    s = {"x": randn(g, m, k, dtype=BF16), "a": randn(g, slots, rank, k, std=k ** -0.5, dtype=BF16),
         "b": randn(g, slots, n, rank, std=0.2, dtype=BF16),
         "scaling": 0.25 + torch.rand(slots, generator=g, device=DEV),
         "bias": randn(g, n, dtype=BF16) if bias else None, "codes": None}
    w = randn(g, n, k, std=0.05)
    if fp8:
        s["codes"], s["scale"] = quantise(s["x"])
        s["w"], s["ws"] = quantise(w)
    else:
        s["w"] = w.to(BF16)
    return s


def call(s, index, **kw):
    args = dict(scaling=s["scaling"], bias=s["bias"])
    args.update(kw)
    if s["codes"] is not None:
        return ops.lora_linear_fp8(s["codes"], s["scale"], s["w"], s["ws"], s["x"], s["a"], s["b"], index, **args)
    return ops.lora_linear(s["x"], s["w"], s["a"], s["b"], index, **args)


def lora_reference(s, owner, scaling=True, bias=True):
    """(y, bound on |call - y|) for int64 owners per row."""
    x = s["x"].double()
    w = s["w"].double()
    base = x
    if s["codes"] is not None:
        w = w * s["ws"].double()[:, None]
        base = s["codes"].double() * s["scale"].double()[:, None]
    y, size = base @ w.t(), base.abs() @ w.abs().t()
    vsize = torch.zeros_like(y)
    for a in range(s["a"].shape[0]):
        at = torch.nonzero(owner == a).flatten()
        if at.numel():
            f = s["scaling"][a].double() if scaling and s["scaling"] is not None else 1.0
            A, B = s["a"][a].double(), s["b"][a].double()
            y[at] += f * (x[at] @ A.t()) @ B.t()
            vsize[at] += f * (x[at].abs() @ A.abs().t()) @ B.abs().t()
    if bias and s["bias"] is not None:
        y += s["bias"].double()
        size += s["bias"].double().abs()
    k, rank = x.shape[1], s["a"].shape[1]
    # the projection: k / 16 tensor-core steps, up to 8 parts, two scales, a bias;
    # the adapter: k / 16 steps and 8 parts for V, 2^-17 for the pair that holds
    # it, then rank / 8 steps
    steps = k / 16 + rank / 8 + 24
    tol = y.abs() * 2.0 ** -8 + size * steps * 2.0 ** -22 + vsize * (2 * steps * 2.0 ** -22 + 2.0 ** -17) + 1e-30
    return y, tol


def owners(index, m, slots, per=1):
    o = index.long().repeat_interleave(per)[:m]
    return torch.where((o >= 0) & (o < slots), o, -1)


def check_lora(s, index, per=1, **kw):
    y, tol = lora_reference(s, owners(index, s["x"].shape[0], s["a"].shape[0], per))
    out = call(s, index, rows_per_index=per, **kw)
    assert out.dtype == BF16
    err = (out.double() - y).abs()
    assert (err <= tol).all(), f"worst {float((err / tol).max()):.2f} of the bound"
    return out


def runs(seed, m, requests, slots):
    """Ragged requests, some without an adapter."""
    g = torch.Generator().manual_seed(seed)
    cuts = [0] + sorted(torch.randint(0, m + 1, (requests - 1,), generator=g).tolist()) + [m]
    ids = torch.randint(-1, slots, (requests,), generator=g)
    return torch.repeat_interleave(ids, torch.tensor([b - a for a, b in zip(cuts, cuts[1:])])).to(torch.int32).to(DEV)


SHAPES = [  # rows, k, n, rank, slots
    (1, 64, 64, 8, 1), (1, 1024, 1024, 16, 3), (2, 8, 1, 8, 2), (16, 256, 136, 24, 16), (17, 1000, 130, 16, 20),
    (31, 72, 257, 40, 4), (33, 1024, 640, 64, 33), (64, 2624, 1024, 16, 64), (65, 256, 384, 32, 7),
    (96, 1024, 1543, 72, 9), (129, 520, 127, 128, 3), (300, 1024, 2000, 256, 5), (777, 1000, 1543, 24, 5),
    (1536, 2624, 1024, 32, 8), (2000, 96, 5248, 8, 300),
]


@pytest.mark.parametrize("m, k, n, rank, slots", SHAPES)
@pytest.mark.parametrize("fp8", [False, True])
def test_lora_linear(m, k, n, rank, slots, fp8):
    if fp8:
        k = (k + 15) // 16 * 16
    s = make(m + n, m, k, n, rank, slots, fp8, bias=m % 2 == 0)
    check_lora(s, runs(m, m, max(1, min(m, 12)), slots))                                  # requests
    g = torch.Generator().manual_seed(m)
    check_lora(s, torch.randint(-2, slots + 2, (m,), generator=g).to(torch.int32).to(DEV))  # every row its own
    check_lora(s, torch.full((m,), slots - 1, dtype=torch.int32, device=DEV))              # one for all
    none = torch.full((m,), -1, dtype=torch.int32, device=DEV)
    base = check_lora(s, none)                                                             # none at all
    far = torch.full((m,), 2 ** 31 - 1, dtype=torch.int32, device=DEV)
    assert torch.equal(base, check_lora(s, far))
    assert ops.op_status() == 0


@pytest.mark.parametrize("fp8", [False, True])
def test_lora_linear_views(fp8):
    m, k, n, rank, slots = 70, 256, 200, 16, 4
    s = make(3, m, k, n, rank, slots, fp8)
    # rows of wider matrices, a weight that is part of a fused one, three axes
    wide = torch.zeros(m, 3 * k, dtype=BF16, device=DEV)
    wide[:, k:2 * k] = s["x"]
    s["x"] = wide[:, k:2 * k]
    fused = torch.zeros(n + 40, k + 64, dtype=torch.uint8 if fp8 else BF16, device=DEV)
    w = s["w"].view(torch.uint8) if fp8 else s["w"]
    fused[20:20 + n, 16:16 + k] = w
    s["w"] = fused[20:20 + n, 16:16 + k].view(s["w"].dtype)
    per = torch.tensor([2, -1, 0, 3, 9], dtype=torch.int32, device=DEV)
    ref = check_lora(s, per, per=16)
    for pad in (0, 1, 4, 8):  # into odd and even strides; nothing beside the rows is touched
        out = torch.full((m, n + 3 + pad), 5.0, dtype=BF16, device=DEV)
        got = call(s, per, rows_per_index=16, out=out[:, 2:2 + n])
        assert got.data_ptr() == out[:, 2:].data_ptr() and torch.equal(out[:, 2:2 + n], ref)
        assert (out[:, :2] == 5).all() and (out[:, 2 + n:] == 5).all()
    s["x"] = s["x"].contiguous().view(7, 10, k)
    if fp8:
        s["codes"], s["scale"] = s["codes"].view(7, 10, k), s["scale"].view(7, 10)
    assert torch.equal(call(s, per, rows_per_index=16), ref.view(7, 10, n))
    s["scaling"] = None
    flat = dict(s, x=s["x"].view(m, k), codes=s["codes"].view(m, k) if fp8 else None,
                scale=s["scale"].view(m) if fp8 else None)
    check_lora(flat, per, per=16)
    assert call(dict(s, x=s["x"][:0], codes=None, w=torch.zeros(n, k, dtype=BF16, device=DEV)), per[:0]).shape == (0, 10, n)


def test_requests_do_not_reach_each_other():
    """A NaN or an infinity in one row, or in one adapter's A, stays in the
    rows it belongs to."""
    m, k, n, rank, slots = 150, 512, 300, 16, 5
    s = make(11, m, k, n, rank, slots)
    index = runs(4, m, 9, slots)
    index[::7] = 2
    clean = check_lora(s, index)
    x = s["x"].clone()
    x[17, 3], x[40, 100] = float("nan"), float("inf")
    got = call(dict(s, x=x), index)
    others = torch.ones(m, dtype=torch.bool, device=DEV)
    others[[17, 40]] = False
    assert torch.equal(got[others], clean[others]) and got[17].isnan().all() and not got[40].isfinite().any()
    a = s["a"].clone()
    a[2, 5, 9] = float("nan")
    got = call(dict(s, a=a), index)
    assert torch.equal(got[index != 2], clean[index != 2]) and got[index == 2].isnan().all()
    # scaling 0 turns an adapter off
    zero = s["scaling"].clone()
    zero[2] = 0
    off = torch.where(index == 2, -1, index).to(torch.int32)
    assert torch.equal(call(s, index, scaling=zero)[index == 2], call(s, off)[index == 2])


def test_lora_linear_many_rows():
    """An output past 2^31 elements."""
    m, k, n = (1 << 19) + 5, 64, 4104
    s = make(12, m, k, n, 8, 3)
    index = (torch.arange(m, device=DEV) % 5 - 1).to(torch.int32)
    out = call(s, index)
    at = torch.tensor([0, 1, (1 << 31) // n, (1 << 31) // n + 1, m - 2, m - 1], device=DEV)
    y, tol = lora_reference(dict(s, x=s["x"][at]), owners(index, m, 3)[at])
    assert ((out[at].double() - y).abs() <= tol).all()


def test_streams_graphs_and_repeats():
    m, k, n, rank, slots = 40, 512, 640, 16, 6
    s1, s2 = make(21, m, k, n, rank, slots), make(22, m, k, n, rank, slots, fp8=True)
    index = runs(3, m, 6, slots)
    w = torch.ones(n, device=DEV)
    ref1, ref2 = check_lora(s1, index), check_lora(s2, index)
    h0 = randn(gen(2), m, n)
    y0 = ops.rms_norm(ref1, w, residual=h0.clone())
    for _ in range(3):  # the same bits each time
        assert torch.equal(call(s1, index), ref1) and torch.equal(call(s2, index), ref2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call(s1, index)
        y = ops.rms_norm(got, w, residual=h0.clone())
    side.synchronize()
    assert torch.equal(got, ref1) and torch.equal(y, y0)
    # two graphs that run at the same time, replayed with new inputs
    torch.cuda.synchronize()
    graphs, outs, h = [], [], h0.clone()
    for s in (s1, s2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = call(s, index)
            outs.append((o, ops.rms_norm(o, w)))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0][0], ref1) and torch.equal(outs[1][0], ref2)
    assert torch.equal(outs[0][1], ops.rms_norm(ref1, w)) and torch.equal(outs[1][1], ops.rms_norm(ref2, w))
    s1["x"].copy_(randn(gen(99), m, k, dtype=BF16))
    index.copy_(runs(8, m, 4, slots))
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0][0], check_lora(s1, index))


def test_block_of_both():
    """Norm, FP8 projection with adapters, norm, projection back: each stage
    against the definition on the stage before it, over an odd batch."""
    m, d, f, slots = 203, 512, 1000, 5
    g = gen(31)
    h = randn(g, m, d, std=2.0)
    delta = randn(g, m, d, dtype=BF16)
    w1, w2 = 1 + randn(g, d, std=0.1), 1 + randn(g, f, std=0.1)
    up, down = make(32, m, d, f, 16, slots, fp8=True), make(33, m, f, d, 24, slots)
    index = runs(5, m, 7, slots)
    h_ref = h + delta.float()
    codes, scale, rows = ops.rms_norm_quant(delta, w1, residual=h, rows=True)
    assert torch.equal(h, h_ref)
    s = dict(up, x=rows, codes=codes, scale=scale)
    mid = check_lora(s, index)
    act = ops.rms_norm(mid, w2)
    back = check_lora(dict(down, x=act), index)
    out = ops.rms_norm(back, w1, residual=h, dtype=F32)
    _, ref = rms_reference(back, w1, 1e-5, h_ref)
    assert ((out.double() - ref).abs() <= y_bound(ref, F32)).all()
    assert torch.equal(h, h_ref + back.float()) and ops.op_status() == 0


def test_gpu_refusals():
    s = make(41, 4, 64, 32, 8, 2)
    index = torch.zeros(4, dtype=torch.int32, device=DEV)
    bad = [dict(s, w=s["w"].cpu()), dict(s, scaling=s["scaling"].cpu()), dict(s, x=s["x"].clone().requires_grad_())]
    for b in bad:
        with pytest.raises(ValueError):
            call(b, index)
    with torch.no_grad():
        assert torch.equal(call(bad[2], index), call(s, index))
    with pytest.raises(ValueError):
        call(s, index, out=s["x"][:, :32])  # overlaps x
    with pytest.raises(ValueError):
        call(s, index, out=torch.empty(4, 33, dtype=BF16, device=DEV))
    with pytest.raises(RuntimeError, match="16-byte"):
        call(dict(s, x=torch.zeros(4, 68, dtype=BF16, device=DEV)[:, 4:]), index)
    x = randn(gen(1), 4, 64)
    with pytest.raises(ValueError):
        ops.rms_norm(x, residual=x)
    with pytest.raises(ValueError):
        ops.rms_norm(x, residual=torch.zeros(64, device=DEV).expand(4, 64))
    with pytest.raises(ValueError):
        ops.rms_norm(x[:2], out=x[1:3])


@pytest.mark.parametrize("m, k, n, rank, slots", [
    (64, 64, 40000, 24, 64),    # more feature tiles than CTAs: K is not split, a CTA stores all rows
    (64, 512, 300, 256, 64), (8, 1024, 512, 136, 8), (13, 2624, 130, 248, 2),
    (9, 20000, 72, 8, 3),       # a long K
    (64, 4096, 130, 64, 9), (50, 2624, 257, 104, 50),  # V by tiles instead of single products
    (48, 1024, 1024, 8, 200), (5, 16, 1, 16, 2), (64, 16, 8, 8, 1),
    (65, 512, 40, 256, 65), (256, 64, 129, 16, 200), (257, 80, 300, 40, 2), (1023, 4096, 520, 48, 31),
])
@pytest.mark.parametrize("fp8", [False, True])
def test_lora_linear_corners(m, k, n, rank, slots, fp8):
    if fp8:
        k = (k + 15) // 16 * 16
    s = make(m * 3 + n, m, k, n, rank, slots, fp8, bias=n % 2 == 0)
    check_lora(s, (torch.arange(m, device=DEV) % slots).to(torch.int32))
    check_lora(s, runs(m + 1, m, max(1, min(m, 9)), slots))
    check_lora(s, torch.tensor([slots - 1, -1, 0], dtype=torch.int32, device=DEV).repeat(m)[:(m + 6) // 7].contiguous(),
               per=7)
    assert ops.op_status() == 0


@pytest.mark.parametrize("m", [1, 7, 24, 64])
@pytest.mark.parametrize("fp8", [False, True])
def test_few_requests_do_not_reach_each_other(m, fp8):
    k, n, rank, slots = 256, 300, 24, 5
    s = make(50 + m, m, k, n, rank, slots, fp8)
    index = (torch.arange(m, device=DEV) // 3 % slots).to(torch.int32)
    clean = check_lora(s, index)
    x = s["x"].clone()
    x[m // 2, 3], x[m - 1, 100] = float("nan"), float("inf")
    got = call(dict(s, x=x), index)
    others = torch.ones(m, dtype=torch.bool, device=DEV)
    others[[m // 2, m - 1]] = False
    assert torch.equal(got[others], clean[others]) and not got[~others].isfinite().any()
    a = s["a"].clone()
    a[0, 5, 9] = float("nan")
    got = call(dict(s, a=a), index)
    assert torch.equal(got[index != 0], clean[index != 0]) and got[index == 0].isnan().all()
    # a slot that nobody uses may hold anything
    a, b = s["a"].clone(), s["b"].clone()
    a[1], b[1] = float("nan"), float("inf")
    other = torch.where(index == 1, 2, index).to(torch.int32)
    assert torch.equal(call(dict(s, a=a, b=b), other), call(s, other))


@pytest.mark.parametrize("rows, d", [(3, 16), (40, 17), (33, 23), (1, 31), (700, 127), (2001, 435), (64, 1001),
                                     (900, 2623), (700, 4001), (5, 4099), (300, 16383), (10000, 129)])
@pytest.mark.parametrize("x_type, r_type", [(BF16, F32), (BF16, BF16), (F32, None)])
def test_rms_norm_odd_rows(rows, d, x_type, r_type):
    """Rows off the 16-byte boundaries: all buffers alike, and not."""
    g = gen(rows + d)
    w = 1 + randn(g, d + 1, std=0.2)
    for lo, ld in ((0, d), (0, d + d % 8), (3, (d + 15) // 8 * 8 + 5)):
        x = randn(g, rows, ld + lo, dtype=x_type)[:, lo:lo + d]
        if r_type is None:
            r = None
        else:
            whole = randn(g, rows, ld + lo, std=3.0, dtype=r_type)
            r, before = whole[:, lo:lo + d], whole.clone()
        _, ref = rms_reference(x, w[:d], 1e-5, r)
        out = torch.full((rows, ld + lo), 9.0, dtype=x_type, device=DEV)
        ops.rms_norm(x, w[:d], residual=r, out=out[:, lo:lo + d])
        assert ((out[:, lo:lo + d].double() - ref).abs() <= y_bound(ref, x_type)).all()
        assert (out[:, :lo] == 9).all() and (out[:, lo + d:] == 9).all()
        if r is not None:
            before[:, lo:lo + d] = (before[:, lo:lo + d].float() + x.float()).to(r_type)
            assert torch.equal(whole, before)
        # the others' rows at distances of their own, a weight off its boundary
        check_rms(x, w[1:], None if r is None else r.clone(), True)


def test_two_streams_at_once():
    """Calls of every kernel in flight on two streams."""
    cases = [make(60 + i, *c) for i, c in enumerate(
        ((1, 512, 256, 16, 2), (64, 1024, 512, 256, 6), (64, 512, 1000, 16, 64), (300, 512, 520, 64, 7)))]
    cases += [make(70, 48, 512, 256, 16, 5, True), make(71, 500, 512, 256, 16, 5, True)]
    index = [(torch.arange(s["x"].shape[0], device=DEV) % s["a"].shape[0]).to(torch.int32) for s in cases]
    refs = [check_lora(s, i) for s, i in zip(cases, index)]
    norm = [ops.rms_norm(r) for r in refs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], ([], [])
    for _ in range(10):
        for j, (s, i) in enumerate(zip(cases, index)):
            for side, st in enumerate(streams):
                with torch.cuda.stream(st):
                    y = call(s, i)
                    got[side].append((j, y, ops.rms_norm(y)))
    torch.cuda.synchronize()
    for j, y, z in got[0] + got[1]:
        assert torch.equal(y, refs[j]) and torch.equal(z, norm[j])
    assert ops.op_status() == 0


FIRST_IN_CAPTURE = """
import sys, torch
sys.path.insert(0, sys.argv[1])
from laya_b200 import ops
which = sys.argv[2]
dev = torch.device("cuda")
m = {"few": 5, "tiles": 64, "many": 300, "rms": 5}[which]
x = torch.ones(m, 1024, dtype=torch.bfloat16, device=dev)
w = torch.ones(64, 1024, dtype=torch.bfloat16, device=dev)
a = torch.ones(2, 256, 1024, dtype=torch.bfloat16, device=dev)
b = torch.ones(2, 64, 256, dtype=torch.bfloat16, device=dev)
i = torch.zeros(m, dtype=torch.int32, device=dev)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y = ops.rms_norm(x) if which == "rms" else ops.lora_linear(x, w, a, b, i)
g.replay()
torch.cuda.synchronize()
want = 1.0 if which == "rms" else 1024 + 256 * 1024
assert (y.float() - want).abs().max() <= want / 256, y
"""


@pytest.mark.parametrize("which", ["few", "tiles", "many", "rms"])
def test_first_call_inside_a_capture(which):
    import pathlib
    import subprocess
    import sys

    root = str(pathlib.Path(ops.__file__).resolve().parents[1])
    done = subprocess.run([sys.executable, "-c", FIRST_IN_CAPTURE, root, which], capture_output=True, text=True,
                          timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


@pytest.mark.parametrize("rows, d", [(5, 64), (300, 72), (40, 1001)])
def test_columns_of_one_buffer(rows, d):
    """x, residual and output as columns of the same rows; what overlaps is refused."""
    g = gen(80 + rows)
    ld = 3 * d + 8 + (-3 * d) % 8
    buffer = randn(g, rows, ld, dtype=BF16)
    before = buffer.clone()
    x, r, out = buffer[:, :d], buffer[:, d:2 * d], buffer[:, 2 * d + 1:3 * d + 1]
    h, y = rms_reference(x, None, 1e-5, r)
    ops.rms_norm(x, residual=r, out=out)
    assert torch.equal(x, before[:, :d]) and torch.equal(r, h.float().to(BF16))
    assert ((out.double() - y).abs() <= y_bound(y, BF16)).all()
    assert torch.equal(buffer[:, 2 * d], before[:, 2 * d]) and torch.equal(buffer[:, 3 * d + 1:], before[:, 3 * d + 1:])
    for lo in (1, d - 1, d + 1, 2 * d - 1):  # beside r's columns, partly over them
        with pytest.raises(ValueError, match="overlaps"):
            ops.rms_norm(buffer[:, lo:lo + d], residual=r)
    with pytest.raises(ValueError, match="overlaps"):  # other rows' strides
        ops.rms_norm(buffer.view(-1)[:rows * d].view(rows, d), residual=r)
    if d % 8:
        return
    n = 24
    s = make(90 + rows, rows, d, n, 16, 3)
    buffer[:, :d] = s["x"]
    s["x"] = buffer[:, :d]
    index = (torch.arange(rows, device=DEV) % 4 - 1).to(torch.int32)
    ref = check_lora(s, index)
    assert torch.equal(call(s, index, out=buffer[:, d:d + n]), ref) and torch.equal(buffer[:, :d], s["x"])
    with pytest.raises(ValueError, match="overlaps"):
        call(s, index, out=buffer[:, d - 1:d - 1 + n])


@pytest.mark.parametrize("m, k, n, rank, slots", [(65, 64, 13000, 8, 3), (257, 512, 5000, 72, 40),
                                                  (130, 256, 9001, 24, 130), (2000, 264, 1290, 40, 9),
                                                  (6500, 2624, 1024, 16, 16)])
@pytest.mark.parametrize("fp8", [False, True])
def test_lora_linear_many_tiles(m, k, n, rank, slots, fp8):
    """More tiles than the kernel for few of them takes: indices of every kind,
    into strided outputs, and with values that are not finite."""
    if fp8:
        k = (k + 15) // 16 * 16
    s = make(m * 5 + n, m, k, n, rank, slots, fp8, bias=n % 2 == 1)
    index = runs(m, m, min(m, 30), slots)
    ref = check_lora(s, index)
    check_lora(s, (torch.arange(m, device=DEV) % slots).to(torch.int32))
    check_lora(s, torch.full((m,), -1, dtype=torch.int32, device=DEV))
    for pad in (0, 1, 5):
        out = torch.full((m, n + 3 + pad), 5.0, dtype=BF16, device=DEV)
        call(s, index, out=out[:, 2:2 + n])
        assert torch.equal(out[:, 2:2 + n], ref) and (out[:, :2] == 5).all() and (out[:, 2 + n:] == 5).all()
    index[::9] = slots - 1
    ref = check_lora(s, index)
    x, a = s["x"].clone(), s["a"].clone()
    x[m // 2, 3], x[m - 1, k // 2] = float("nan"), float("inf")
    got = call(dict(s, x=x), index)
    others = torch.ones(m, dtype=torch.bool, device=DEV)
    others[[m // 2, m - 1]] = False
    assert torch.equal(got[others], ref[others])
    a[slots - 1, 5, 9] = float("nan")
    got = call(dict(s, a=a), index)
    mine = index == slots - 1
    assert torch.equal(got[~mine], ref[~mine]) and got[mine].isnan().all()
    assert ops.op_status() == 0


def test_first_and_last_rows_of_row_tiles():
    """Rows behind the last one are left as they were."""
    for m in (63, 64, 65, 127, 129, 192, 193, 255, 257):
        s = make(m, m, 128, 40, 16, 5)
        whole = torch.full((m + 70, 40), 3.0, dtype=BF16, device=DEV)
        index = (torch.arange(m, device=DEV) % 6 - 1).to(torch.int32)
        ref = check_lora(s, index)
        call(s, index, out=whole[1:m + 1])
        assert torch.equal(whole[1:m + 1], ref) and (whole[0] == 3).all() and (whole[m + 1:] == 3).all()


@pytest.mark.parametrize("m, k, n, rank, slots", [(64, 4096, 130, 128, 9), (37, 8192, 72, 200, 37), (64, 2048, 257, 256, 64),
                                                  (64, 16384, 40, 24, 64), (33, 40000, 24, 16, 5), (64, 24000, 16, 32, 3),
                                                  (64, 40968, 33, 8, 64), (64, 65536, 16, 8, 64),
                                                  (61, 42000, 24, 24, 61)])
def test_few_rows_of_much_work(m, k, n, rank, slots):
    """V of up to 64 rows by tiles."""
    s = make(m + rank, m, k, n, rank, slots, bias=n % 2 == 0)
    check_lora(s, (torch.arange(m, device=DEV) % slots).to(torch.int32))
    check_lora(s, runs(m + 3, m, 9, slots))
    check_lora(s, torch.zeros(m, dtype=torch.int32, device=DEV))
    assert ops.op_status() == 0
