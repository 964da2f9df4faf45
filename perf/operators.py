"""The row operators of laya_b200.ops as work to be measured: one pass through
each over the sizes that a server of the Laya network, or of a block built
beside it, meets.

Two operators, which a block runs one after the other: ``rms`` adds a
projection's output to the residual stream, normalises the sum and (with
``codes``) writes it as e4m3 codes with a scale per row; ``lora`` is the
projection that reads those rows, with the low-rank adapters of all the
requests of the batch beside the shared weight, in bf16 or (``fp8``) on the
e4m3 operand.

A case is a dict of plain values; ``run`` makes one pass, either by the plain
form below (``own`` false: elementary torch operations in 32 bits, rounded
once) or by the framework's call (``own`` true).
"""
import math
import sys
from pathlib import Path

import torch

own = False

PACKAGE = str(Path(__file__).resolve().parents[1] / "laya-inference-engine_b200")

E4M3_MAX = 448.0
EPS = 1e-5
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _ops():
    if PACKAGE not in sys.path:
        sys.path.insert(0, PACKAGE)
    from laya_b200 import ops
    return ops


# ------------------------------------------------------------------- cases
def _lora(name, rows, k, n, rank, adapters, requests, fp8=False, bias=False):
    return {"name": name, "op": "lora", "rows": rows, "k": k, "n": n, "rank": rank, "adapters": adapters,
            "requests": requests, "fp8": fp8, "bias": bias}


def _rms(name, rows, d, x="bf16", residual="f32", codes=False, keep=True):
    return {"name": name, "op": "rms", "rows": rows, "d": d, "x": x, "residual": residual, "codes": codes,
            "keep": keep}


def listed():
    return [
        # the smallest call: one row of one request (the scorer's width)
        _lora("lora_row", 1, 1024, 1024, 16, 1, 1),
        # single rows of 64 requests, each with an adapter of its own, into the GEGLU projection
        _lora("lora_64_requests", 64, 1024, 5248, 16, 64, 64),
        # 16 questions of about 96 tokens, eight tenants, back from the GEGLU width
        _lora("lora_16_questions", 1536, 2624, 1024, 32, 8, 16),
        # odd sizes: ragged requests, a width that ends inside every tile, a rank that is no power of two
        _lora("lora_ragged", 777, 1000, 1543, 24, 5, 11, bias=True),
        # a full batch of 64 questions, up to 512 tokens each, 32 tenants with a wide adapter
        _lora("lora_64_questions", 8192, 1024, 5248, 64, 32, 64),
        # the same 64 single rows on the FP8 operand
        _lora("lora_64_requests_fp8", 64, 1024, 5248, 16, 64, 64, fp8=True),
        # a full batch on the FP8 operand, back from the GEGLU width
        _lora("lora_64_questions_fp8", 8192, 2624, 1024, 16, 16, 64, fp8=True),
        # one row into the residual stream, codes and rows kept: the operand of an FP8 projection with adapters
        _rms("rms_row", 1, 1024, codes=True),
        # 16 questions of 96 tokens, as the projection above reads them
        _rms("rms_16_questions", 1536, 1024, codes=True),
        # an odd width in fp32, no residual stream: a final norm
        _rms("rms_odd_f32", 1237, 2623, x="f32", residual="none"),
        # a full batch, codes alone: the operand of an FP8 projection without adapters
        _rms("rms_64_questions_codes", 32768, 1024, codes=True, keep=False),
        # a wide block in bf16 throughout
        _rms("rms_wide", 16384, 4096, residual="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _plain_cost(c):
    return c["rows"] * (c["k"] * c["n"] + c["adapters"] * c["rank"] * (c["k"] + c["n"]))


def draw(rng):
    if rng.random() < 0.6:
        most = max(_plain_cost(c) for c in listed() if c["op"] == "lora")
        while True:
            rows = _log(rng, 1, 8192)
            requests = rng.choice([rows, _log(rng, 1, 64)]) if rows <= 256 else _log(rng, 1, 64)
            requests = min(rows, requests)
            fp8 = rng.random() < 0.4
            c = _lora("", rows, 16 * _log(rng, 12, 164) + (0 if fp8 else rng.choice([0, 8])), _log(rng, 190, 5250),
                      8 * rng.choice([1, 2, 2, 3, 4, 5, 8, 8, 12, 16]), min(requests, _log(rng, 1, 64)), requests,
                      fp8=fp8, bias=rng.random() < 0.3)
            if _plain_cost(c) <= most:
                break
    else:
        rows, d = _log(rng, 1, 32768), _log(rng, 64, 8192)
        if rng.random() < 0.6:
            d = max(64, d // 64 * 64)
        rows = max(1, min(rows, 16384 * 4096 // d))
        codes = rng.random() < 0.6
        c = _rms("", rows, d, x=rng.choice(["bf16", "bf16", "f32"]), residual=rng.choice(["f32", "f32", "bf16", "none"]),
                 codes=codes, keep=not codes or rng.random() < 0.5)
    del c["name"]
    return c


def _served(c):
    """(requests with an adapter, rows they hold on average)."""
    none = c["requests"] // 8
    return c["requests"] - none, c["rows"] * (c["requests"] - none) / c["requests"]


def work(c):
    if c["op"] == "rms":
        size = {"bf16": 2, "f32": 4, "none": 0}
        per = size[c["x"]] + 2 * size[c["residual"]] + (size[c["x"]] if c["keep"] else 0) + (1 if c["codes"] else 0)
        e = c["rows"] * c["d"]
        return {"bytes": e * per + c["d"] * 4 + (c["rows"] * 4 if c["codes"] else 0), "flops": 6 * e}
    m, k, n, r = c["rows"], c["k"], c["n"], c["rank"]
    requests, rows = _served(c)
    used = min(c["adapters"], requests)
    base = (m + n) * k * (1 if c["fp8"] else 2) + ((m + n) * 4 + m * k * 2 if c["fp8"] else 0)
    return {"bytes": base + m * n * 2 + used * r * (k + n) * 2 + m * 4 + (n * 2 if c["bias"] else 0),
            "flops": 2 * m * n * k + 2 * rows * r * (k + n)}


# ------------------------------------------------------------------ inputs
def _index(c, seed, device):
    """int32 [rows]: the adapter of each row; a request's rows follow one
    another, one request in eight has none, every adapter is used by one of
    the others while there are enough of them."""
    g = torch.Generator().manual_seed(seed * 2 + 1)
    m, q = c["rows"], c["requests"]
    cuts = torch.sort(torch.randperm(m - 1, generator=g)[:q - 1] + 1).values if q > 1 else torch.empty(0, dtype=torch.long)
    lengths = torch.diff(torch.cat([torch.zeros(1, dtype=torch.long), cuts, torch.full((1,), m)]))
    ids = torch.arange(q) % c["adapters"]
    ids[q - q // 8:] = -1
    ids = ids[torch.randperm(q, generator=g)]
    return torch.repeat_interleave(ids, lengths).to(torch.int32).to(device)


def _rows_e4m3(x):
    """e4m3 codes of the rows of x and their scales (amax / 448)."""
    scale = (x.abs().amax(dim=1) / E4M3_MAX).clamp_min(1e-12)
    return (x / scale[:, None]).to(torch.float8_e4m3fn), scale


def prepare(c, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=g, device=dev) * std

    if c["op"] == "rms":
        x = normal(c["rows"], c["d"], std=0.5).to(TYPES[c["x"]])
        # a residual stream: rows of different size, a few channels much larger than the rest
        h = None
        if c["residual"] != "none":
            h = normal(c["rows"], c["d"]) * torch.exp(normal(c["rows"], 1))
            h[:, ::97] *= 8
            h = h.to(TYPES[c["residual"]])
        return {"case": c, "x": x, "residual": h, "weight": 1 + normal(c["d"], std=0.1)}
    m, k, n, r, s = c["rows"], c["k"], c["n"], c["rank"], c["adapters"]
    x = normal(m, k).to(torch.bfloat16)
    w = normal(n, k, std=0.02)
    state = {"case": c, "x": x, "lora_a": normal(s, r, k, std=k ** -0.5).to(torch.bfloat16),
             "lora_b": normal(s, n, r, std=0.02).to(torch.bfloat16),
             "scaling": 0.5 + 2 * torch.rand(s, generator=g, device=dev),
             "index": _index(c, seed, dev), "bias": normal(n, std=0.02).to(torch.bfloat16) if c["bias"] else None}
    if c["fp8"]:
        state["codes"], state["scale"] = _rows_e4m3(x.float())
        state["weight"], state["weight_scale"] = _rows_e4m3(w)
    else:
        state["weight"] = w.to(torch.bfloat16)
    return state


# ------------------------------------------------------------- the operators
def _plain_rms(s):
    """h += x; y = h / sqrt(mean(h^2) + eps) * w; codes = e4m3(y / scale),
    scale = max|y| / 448."""
    c = s["case"]
    h = s["x"].float()
    out = {}
    if s["residual"] is not None:
        h = h + s["residual"].float()
        s["residual"].copy_(h)
        out["residual"] = s["residual"]
    y = h * torch.rsqrt(h.square().mean(dim=1, keepdim=True) + EPS) * s["weight"]
    if c["codes"]:
        out["codes"], out["scale"] = _rows_e4m3(y)
    if c["keep"]:
        out["y"] = y.to(s["x"].dtype)
    return out


def _plain_lora(s):
    """y = x W^T + bias + scaling_a (x A_a^T) B_a^T, a the row's adapter."""
    c = s["case"]
    x, slots, rank = s["x"].float(), c["adapters"], c["rank"]
    if c["fp8"]:
        y = (s["codes"].float() * s["scale"][:, None]) @ (s["weight"].float() * s["weight_scale"][:, None]).t()
    else:
        y = x @ s["weight"].float().t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    mine = (s["index"][:, None] == torch.arange(slots, device=x.device)[None, :]).float() * s["scaling"][None, :]
    v = (x @ s["lora_a"].float().reshape(slots * rank, -1).t()).view(-1, slots, rank) * mine[:, :, None]
    b = s["lora_b"].float().permute(0, 2, 1).reshape(slots * rank, -1)
    return (y + v.reshape(-1, slots * rank) @ b).to(torch.bfloat16)


def _own_rms(s):
    ops, c, out = _ops(), s["case"], {}
    if c["codes"]:
        r = ops.rms_norm_quant(s["x"], s["weight"], eps=EPS, residual=s["residual"], rows=c["keep"])
        out["codes"], out["scale"] = r[0], r[1]
        if c["keep"]:
            out["y"] = r[2]
    else:
        out["y"] = ops.rms_norm(s["x"], s["weight"], eps=EPS, residual=s["residual"])
    if s["residual"] is not None:
        out["residual"] = s["residual"]
    return out


def _own_lora(s):
    ops = _ops()
    if s["case"]["fp8"]:
        return ops.lora_linear_fp8(s["codes"], s["scale"], s["weight"], s["weight_scale"], s["x"], s["lora_a"],
                                   s["lora_b"], s["index"], scaling=s["scaling"], bias=s["bias"])
    return ops.lora_linear(s["x"], s["weight"], s["lora_a"], s["lora_b"], s["index"], scaling=s["scaling"],
                           bias=s["bias"])


def run(s):
    if s["case"]["op"] == "rms":
        return _own_rms(s) if own else _plain_rms(s)
    return _own_lora(s) if own else _plain_lora(s)


# -------------------------------------------------------- the definition, 64 bits
def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "rms":
        h = s["x"].double()
        out = {}
        if s["residual"] is not None:
            h = h + s["residual"].double()
            out["residual"] = h
        y = h / torch.sqrt((h * h).sum(dim=1, keepdim=True) / c["d"] + EPS) * s["weight"].double()
        if c["codes"]:
            out["scale"] = y.abs().max(dim=1).values / E4M3_MAX
            out["codes"] = y / out["scale"][:, None]
        if c["keep"]:
            out["y"] = y
        return out
    w = s["weight"].double()
    rows = s["x"].double()
    if c["fp8"]:
        w = w * s["weight_scale"].double()[:, None]
        y = torch.mm(s["codes"].double() * s["scale"].double()[:, None], w.t())
    else:
        y = torch.mm(rows, w.t())
    if s["bias"] is not None:
        y += s["bias"].double()
    for a in range(c["adapters"]):
        at = torch.nonzero(s["index"] == a).flatten()
        low = torch.mm(rows[at], s["lora_a"][a].double().t()) * s["scaling"][a].double()
        y[at] += torch.mm(low, s["lora_b"][a].double().t())
    return y
