"""Every projection of a one-layer network with adapters, in bf16 and FP8, from the
GPU's own stage before it (FP8: its own codes and scales), in 64 bits.

Bounds, from the arithmetic: fp32 sums and the pair that holds V as in
test_gpu_ops; each rounding to bf16 half a step, 2^-8 of the value; where a stage
before is not the GPU's own (the embedding's LayerNorm), the interval that its fp32
error leaves is carried through the bf16 rounding, the codes and the weights.  The
adapters are as large as the shared projection's output, and each stage has to be
outside its bounds for most values when they are left out or exchanged."""
import numpy as np
import pytest
import torch

from laya_b200.config import LayaConfig
from laya_b200.engine import NativeForward
from laya_b200.weights import as_float32, bf16_bits_to_f32, seeded_weights
from laya_b200.workload import pack, synthetic_items
from oracle import laya_oracle as O
from test_gpu_adapters import make_adapter

pytestmark = pytest.mark.gpu

CFG = LayaConfig(layers=1, hidden=256, heads=4, intermediate=384, vocab=1000, pad_token_id=999, max_len=512,
                 head_layers=0, head_heads=4, head_ff=512, act_hidden=64)
RANK = 12
HALF = 2.0 ** -8  # half a bf16 step, of the value


def bf(x):
    return x.float().to(torch.bfloat16).double()


class Rows:
    """A projection's input: x the bf16 rows, base what the shared weight reads, and
    how far both may be off."""

    def __init__(self, x, base=None, dx=None, dbase=None):
        self.x, self.base = x, x if base is None else base
        self.dx = torch.zeros_like(x) if dx is None else dx
        self.dbase = self.dx if base is None else torch.zeros_like(x) if dbase is None else dbase


def norm_rows(y, margin, fp8):
    """Rows from a LayerNorm known to `margin`, and which of them are usable: not
    those whose FP8 scale is uncertain."""
    lo, hi = bf(y - margin), bf(y + margin)
    mid = bf(y)
    sure = torch.ones(y.shape[0], dtype=torch.bool)
    if not fp8:
        return Rows(mid, dx=hi - lo), sure
    a = torch.maximum(lo.abs().amax(1), hi.abs().amax(1))
    sure = torch.minimum(lo.abs(), hi.abs()).amax(1) == a

    def deq(v):
        scale = torch.clamp(a.float()[:, None] * O.INV_E4M3_MAX, min=O.FP8_MIN_SCALE)
        return (O.e4m3(torch.clamp(v.float() / scale, -448, 448)) * scale).double()

    return Rows(mid, deq(mid), hi - lo, deq(hi) - deq(lo)), sure


class Net:
    def __init__(self, weights, adapters, fp8):
        self.w = {k: torch.from_numpy(v).double() for k, v in as_float32(weights).items()}
        self.fp8 = fp8
        if fp8:
            for k in ("wqkv", "wo", "wi", "wo2"):
                q, s = O.fp8_quantize_rows(self.w[f"enc.0.{k}"].float())
                self.w[f"enc.0.{k}"] = q.double() * s.double()
        self.adapters = {nm: ({k: tuple(torch.from_numpy(bf16_bits_to_f32(m)).double() for m in pair)
                               for k, pair in ad.items()}, f) for nm, (ad, f) in adapters.items()}

    def project(self, rows, name, chosen):
        """(x W^T + the questions' adapter terms, bound before the rounding)."""
        w = self.w[name]
        y, size = rows.base @ w.t(), rows.base.abs() @ w.abs().t()
        tol = rows.dbase.abs() @ w.abs().t()
        vsize = torch.zeros_like(y)
        s = y.shape[0] // len(chosen)
        for q, nm in enumerate(chosen):
            if nm is None:
                continue
            pairs, f = self.adapters[nm]
            a, b = pairs[name]
            at = slice(q * s, (q + 1) * s)
            y[at] += f * (rows.x[at] @ a.t()) @ b.t()
            vsize[at] += f * (rows.x[at].abs() @ a.abs().t()) @ b.abs().t()
            tol[at] += f * (rows.dx[at].abs() @ a.abs().t()) @ b.abs().t()
        steps = w.shape[1] / 16 + 2 + 24
        return y, tol + size * steps * 2.0 ** -22 + vsize * (2 * steps * 2.0 ** -22 + 2.0 ** -17)


def rounded(tol, y):
    return tol + HALF * (y.abs() + tol)


def layer_norm(h, dh, w):
    """LayerNorm of h, known to dh, to first order in dh (a tenth on top for the rest)."""
    c = h - h.mean(1, keepdim=True)
    sd = torch.sqrt(c.square().mean(1, keepdim=True) + CFG.norm_eps)
    n = c / sd
    off = (dh + dh.mean(1, keepdim=True) + n.abs() * dh.square().mean(1, keepdim=True).sqrt()) / sd * 1.1
    return n * w, (off + 2.0 ** -20 * (1 + n.abs())) * w.abs()


def stages(net, got, inp, b, s, chosen):
    """name -> (GPU's values, definition, bound, usable rows), with these adapters."""
    T, d, heads = b * s, CFG.hidden, CFG.heads
    w = net.w
    ids = torch.from_numpy(inp["input_ids"]).reshape(-1)
    h0, dh0 = layer_norm(w["embed.tok"][ids], torch.zeros(T, d, dtype=torch.float64), w["embed.norm.w"])
    out = {}
    # QKV with the rotary embedding
    x, sure = norm_rows(h0, dh0, net.fp8)
    y, tol = net.project(x, "enc.0.wqkv", chosen)
    tol = rounded(tol, y)
    cos, sin = (t[:s].double().repeat(b, 1)[:, None, :] for t in O.rope_tables(CFG.rope_theta_global, CFG.max_len, 64))

    def rotate(t, sign):
        halves = t.view(T, heads, 64)
        other = torch.cat((sign * halves[..., 32:], halves[..., :32]), dim=-1)
        return (halves, other)

    ref, bound = [], []
    for part in range(3):
        yp, tp = y[:, part * d:(part + 1) * d], tol[:, part * d:(part + 1) * d]
        if part == 2:
            ref.append(yp)
            bound.append(tp)
            continue
        a, o = rotate(yp, -1.0)
        ta, to = rotate(tp, 1.0)
        r = a * cos + o * sin
        t = (ta * cos.abs() + to * sin.abs()) * (1 + 2.0 ** -20) + 2.0 ** -20 * (a.abs() + o.abs())
        ref.append(r.reshape(T, d))
        bound.append(rounded(t, r).reshape(T, d))
    out["qkv"] = got["qkv"], torch.cat(ref, 1), torch.cat(bound, 1), sure
    every = torch.ones(T, dtype=torch.bool)
    # Wo into the residual, seen through mlp_norm
    y, tol = net.project(Rows(got["attn"], got.get("a8")), "enc.0.wo", chosen)
    h1, dh1 = h0 + y, dh0 + rounded(tol, y)
    n1, dn1 = layer_norm(h1, dh1, w["enc.0.mlp_norm.w"])
    out["wo"] = got["n"], n1, rounded(dn1, n1), every
    # Wi with GEGLU
    y, tol = net.project(Rows(got["n"], got.get("n8")), "enc.0.wi", chosen)
    tol = rounded(tol, y)
    (act, gate), (ta, tg) = y.chunk(2, dim=1), tol.chunk(2, dim=1)
    e = torch.nn.functional.gelu(act)
    te = 1.13 * ta + act.abs() * 2.0 ** -22
    te = rounded(te, e)
    g = e * gate
    out["wi"] = got["g"], g, rounded(e.abs() * tg + gate.abs() * te + te * tg, g), every
    # Wo2 into the residual, seen through final_norm (fp32)
    y, tol = net.project(Rows(got["g"], got.get("g8")), "enc.0.wo2", chosen)
    h2, dh2 = h1 + y, dh1 + rounded(tol, y)
    n2, dn2 = layer_norm(h2, dh2, w["final_norm.w"])
    emb = w["type_emb"][torch.from_numpy(inp["qtype"]).long()].repeat_interleave(s, 0)
    out["wo2"] = got["h"], n2 + emb, dn2 + 2.0 ** -20 * (1 + emb.abs()), every
    return out


@pytest.mark.parametrize("b, s", [(1, 40), (2, 32), (2, 192), (4, 512), (8, 512)])
@pytest.mark.parametrize("precision", ["bf16", "fp8"])
def test_stages(precision, b, s):
    fp8 = precision == "fp8"
    weights = seeded_weights(CFG, seed=3)
    adapters = {nm: (make_adapter(CFG, seed, RANK, size=0.04), f) for seed, nm, f in ((1, "a", 1.5), (2, "b", 2.0))}
    chosen = ["b", "a", None, "b", "a", "a", "b", None][:b]
    items = synthetic_items([s] * b, (["choice", "noul", "score"] * 3)[:b], seed=11, vocab=CFG.vocab)
    inp = pack(items, b, s, 4, CFG.pad_token_id)
    T, d, inter = b * s, CFG.hidden, CFG.intermediate
    nf = NativeForward(0, CFG, weights, precision, max_batch=b, max_options=4)
    try:
        nf.enable_adapters(2, RANK)
        nf.set_adapter(0, *adapters["a"])
        nf.set_adapter(1, *adapters["b"])
        slot = nf.capture_adapters(b, s, 4, True)
        nf.run(slot, inp, np.array([{"a": 0, "b": 1, None: -1}[c] for c in chosen], np.int32))

        def read(name, columns):
            return torch.from_numpy(bf16_bits_to_f32(nf.read_buffer(name, (T, columns), np.uint16))).double()

        got = {"qkv": read("qkv", 3 * d), "attn": read("attn", d), "n": read("n", d), "g": read("g", inter),
               "h": torch.from_numpy(nf.read_buffer("h", (T, d), np.float32)).double()}
        if fp8:
            for name, columns in (("n8", d), ("a8", d), ("g8", inter)):
                codes = torch.from_numpy(nf.read_buffer(name, (T, columns), np.uint8)).view(torch.float8_e4m3fn)
                scale = torch.from_numpy(nf.read_buffer(name + "s", (T,), np.float32))
                got[name] = codes.double() * scale.double()[:, None]
    finally:
        nf.close()
    net = Net(weights, adapters, fp8)
    right = stages(net, got, inp, b, s, chosen)
    none = stages(net, got, inp, b, s, [None] * b)
    other = stages(net, got, inp, b, s, [{"a": "b", "b": "a", None: None}[c] for c in chosen])
    adapted = torch.tensor([c is not None for c in chosen]).repeat_interleave(s)
    for name, (value, ref, bound, sure) in right.items():
        assert float(sure.float().mean()) > 0.8, name
        off = (value - ref).abs()[sure]
        worst = float((off / bound[sure]).max())
        rows = sure & adapted
        seen = [float(((value - x[name][1]).abs() > x[name][2])[rows].float().mean()) for x in (none, other)]
        print(f"{precision} {b}x{s} {name}: {worst:.2f} of the bound; outside it without adapters "
              f"{seen[0]:.0%}, exchanged {seen[1]:.0%}")
        assert worst <= 1, name
        assert min(seen) > 0.5, name
