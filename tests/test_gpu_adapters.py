"""Adapters in the engine's forward on the GPU: batches whose questions run with
different adapters, against the CPU oracle with the adapters added to each
question's projections (fp32, one rounding to bf16, as the other epilogues
round), in bf16 and FP8, over the row counts that take different kernels."""
import threading

import numpy as np
import pytest
import torch

from laya_b200.config import TINY, LayaConfig
from laya_b200.engine import B200Engine, NativeForward, request_from_items
from laya_b200.weights import adapted_projections, as_float32, bf16_bits_to_f32, check_adapter, seeded_weights
from laya_b200.workload import pack, synthetic_items
from oracle import laya_oracle as O

pytestmark = pytest.mark.gpu

# the tolerances of the plain forward (test_gpu_parity): bf16 2e-2, FP8 6e-2
TOL = {"bf16": 2e-2, "fp8": 6e-2}
WIDE = LayaConfig(layers=2, hidden=1024, heads=16, intermediate=640, vocab=1000, pad_token_id=999, max_len=512,
                  head_layers=1, head_heads=16, head_ff=512, act_hidden=64)


def make_adapter(cfg, seed, rank, names=None, size=0.02):
    """Every projection (or `names`), N(0, size) like the weights; rank differs by projection."""
    rng = np.random.Generator(np.random.PCG64(seed))
    out = {}
    for i, (name, (n, k)) in enumerate(adapted_projections(cfg).items()):
        if names is None or name in names:
            r = max(1, rank - i % 3)
            out[name] = (rng.standard_normal((r, k), dtype=np.float32) * np.float32(2 * size),
                         rng.standard_normal((n, r), dtype=np.float32) * np.float32(2 * size))
    return check_adapter(out, cfg)


class AdaptedOracle(O.Oracle):
    """The oracle with an (adapter, scaling) or None per question."""

    def __init__(self, weights, cfg, chosen, precision="bf16"):
        super().__init__(weights, cfg, precision)
        self.chosen = chosen

    def _enc(self, x, name):
        base = O.encoder_linear(x, self.w[name], self.precision, self.qcache, name) if self.precision != "bf16" \
            else x @ self.w[name].t()
        rows = x.shape[0] // len(self.chosen)
        for q, pair in enumerate(self.chosen):
            if pair is not None and name in pair[0]:
                a, b = (torch.from_numpy(bf16_bits_to_f32(m)) for m in pair[0][name])
                part = x[q * rows:(q + 1) * rows]
                base[q * rows:(q + 1) * rows] += pair[1] * (part @ a.t()) @ b.t()
        return O.bf16(base)


def compare(cfg, precision, weights, adapters, lengths, batch, seq, names, slots=4, rank=24):
    """One padded batch through NativeForward; returns (GPU, oracle, unadapted oracle) logits."""
    items = synthetic_items(lengths, ["choice" if n > 4 else "noul" for n in lengths], seed=len(lengths),
                            vocab=cfg.vocab)
    inp = pack(items, batch, seq, 4, cfg.pad_token_id)
    order = list(adapters)
    index = np.full(batch, -1, np.int32)
    for q, nm in enumerate(names):
        if nm is not None:
            index[q] = order.index(nm)
    nf = NativeForward(0, cfg, weights, precision, max_batch=batch, max_options=4)
    try:
        nf.enable_adapters(slots, rank)
        for i, nm in enumerate(order):
            nf.set_adapter(i, adapters[nm][0], adapters[nm][1])
        slot = nf.capture_adapters(batch, seq, 4, False)
        logits, act = nf.run(slot, inp, index)
        again = nf.run(slot, inp, index)
        assert np.array_equal(logits, again[0]) and np.array_equal(act, again[1])
    finally:
        nf.close()
    chosen = [adapters[names[q]] if q < len(names) and names[q] is not None else None for q in range(batch)]
    ref = AdaptedOracle(weights, cfg, chosen, precision).forward(**inp)
    plain = O.Oracle(weights, cfg, precision).forward(**inp)
    mm = inp["marker_mask"].copy()
    mm[len(lengths):] = False
    return (logits, act), ref, plain, mm


CASES = [  # lengths, batch, seq, adapter of each question
    ([64], 1, 64, ["a"]), ([20], 1, 32, ["b"]), ([32, 17], 2, 32, ["b", None]), ([9, 16, 3], 4, 16, ["a", "b", "a"]),
    ([96, 50, 70, 96], 4, 96, ["a", "b", None, "a"]), ([130, 192], 2, 192, [None, "b"]),
    ([512, 300, 64, 90, 400], 8, 512, ["b", None, "a", "a", "c"]), ([65], 1, 96, ["c"]),
]


@pytest.mark.parametrize("lengths, batch, seq, names", CASES)
@pytest.mark.parametrize("precision", ["bf16", "fp8"])
def test_mixed_batch_matches_the_oracle(lengths, batch, seq, names, precision):
    cfg = TINY
    w = seeded_weights(cfg, seed=5)
    adapters = {"a": (make_adapter(cfg, 1, 16), 2.0), "b": (make_adapter(cfg, 2, 7), 4.0),
                "c": (make_adapter(cfg, 3, 24, names=("enc.1.wi", "enc.3.wo2", "enc.0.wqkv")), 3.0)}
    got, ref, plain, mm = compare(cfg, precision, w, adapters, lengths, batch, seq, names)
    n = len(lengths)
    err = np.abs(got[0][mm] - ref[0][mm]).max(), np.abs(got[1][:n] - ref[1][:n]).max()
    assert max(err) <= TOL[precision], err
    moved = np.abs(plain[0] - ref[0])[mm].max()
    print(f"adapted {precision} {batch}x{seq}: logits {err[0]:.3e}, act {err[1]:.3e}, adapters move them {moved:.3e}")
    # the logits of this small random network are small: the adapters' effect on
    # them has to be there, not only within the tolerance
    if precision == "bf16":
        assert err[0] < moved / 2


@pytest.mark.parametrize("precision", ["bf16", "fp8"])
def test_wide_network_takes_the_wide_tiles(precision):
    cfg = WIDE
    w = seeded_weights(cfg, seed=8)
    adapters = {"a": (make_adapter(cfg, 4, 64), 1.0), "b": (make_adapter(cfg, 5, 33), 2.0)}
    lengths = [256, 200, 256, 64, 31, 256, 180, 256, 100, 256]
    names = ["a", "b", None, "a", "a", "b", None, "b", "a", "a"]
    got, ref, plain, mm = compare(cfg, precision, w, adapters, lengths, 16, 256, names, slots=2, rank=64)
    err = np.abs(got[0][mm] - ref[0][mm]).max()
    assert err <= TOL[precision], err


def check_stages(shapes):
    """QKV with the rotary embedding, GEGLU and the residual sums of a one-layer
    network, each from the GPU's own stage before it, to a bf16 step."""
    cfg = LayaConfig(layers=1, hidden=256, heads=4, intermediate=384, vocab=1000, pad_token_id=999, max_len=512,
                     head_layers=0, head_heads=4, head_ff=512, act_hidden=64)
    w = seeded_weights(cfg, seed=3)
    wf = {k: torch.from_numpy(v) for k, v in as_float32(w).items()}
    ad = {nm: (make_adapter(cfg, s, 12), 1.5) for s, nm in ((1, "a"), (2, "b"))}
    for b, s in shapes:
        items = synthetic_items([s] * b, ["choice", "noul"] * (b // 2), seed=11, vocab=cfg.vocab)
        inp = pack(items, b, s, 4, cfg.pad_token_id)
        nf = NativeForward(0, cfg, w, "bf16", max_batch=b, max_options=4)
        try:
            nf.enable_adapters(2, 12)
            nf.set_adapter(0, *ad["a"])
            nf.set_adapter(1, *ad["b"])
            slot = nf.capture_adapters(b, s, 4, True)
            nf.run(slot, inp, np.array([1, 0] * (b // 2), np.int32))
            T, d, inter = b * s, cfg.hidden, cfg.intermediate
            bits = {n: torch.from_numpy(bf16_bits_to_f32(nf.read_buffer(n, (T, c), np.uint16)))
                    for n, c in (("qkv", 3 * d), ("attn", d), ("g", inter))}
        finally:
            nf.close()
        orc = AdaptedOracle(w, cfg, [ad["b"], ad["a"]] * (b // 2))
        ids = torch.from_numpy(inp["input_ids"]).reshape(-1)
        h0 = O.layer_norm(wf["embed.tok"][ids], wf["embed.norm.w"], None, cfg.norm_eps)
        gcos, gsin = O.rope_tables(cfg.rope_theta_global, cfg.max_len, 64)
        r5 = orc._enc(O.bf16(h0), "enc.0.wqkv").view(b, s, 3, cfg.heads, 64)
        qkv = torch.cat([O.rope(r5[:, :, 0], gcos, gsin)[:, :, None], O.rope(r5[:, :, 1], gcos, gsin)[:, :, None],
                         r5[:, :, 2:]], dim=2).reshape(T, 3 * d)
        h1 = h0 + orc._enc(bits["attn"], "enc.0.wo")
        n1 = O.bf16(O.layer_norm(h1, wf["enc.0.mlp_norm.w"], None, cfg.norm_eps))
        act, gate = orc._enc(n1, "enc.0.wi").chunk(2, dim=-1)
        g = O.bf16(O.bf16(O.gelu(act)) * gate)
        # another summation order moves a value across a bf16 rounding border now
        # and then: one step (2^-7 of the value) where it does, few where it may.
        # GEGLU rounds act, gelu and gate first: up to three steps
        for name, ref, steps in (("qkv", qkv, 2), ("g", g, 4)):
            off = (bits[name] - ref).abs()
            assert (off <= steps * 2.0 ** -7 * ref.abs() + 2e-3).all(), (name, float(off.max()))
            assert float((off > 1e-6).float().mean()) < 0.05, name


def test_stages_with_adapters():
    check_stages(((2, 192), (2, 32)))


def test_stages_with_adapters_over_many_tiles():
    """The same on tiles of 256 rows, the residual projections among them."""
    check_stages(((4, 512), (8, 512)))


def test_no_adapter_in_an_adapted_batch():
    """Questions without an adapter, adapters that are zero, and slots that were
    cleared add nothing, and lie within rounding of the plain forward."""
    cfg = TINY
    w = seeded_weights(cfg, seed=6)
    items = synthetic_items([96, 60, 80], ["choice", "noul", "score"], seed=2, vocab=cfg.vocab)
    inp = pack(items, 4, 96, 4, cfg.pad_token_id)
    nf = NativeForward(0, cfg, w, "bf16", max_batch=4, max_options=4)
    try:
        nf.enable_adapters(3, 16)
        plain = nf.run(nf.capture(4, 96, 4, False), inp)
        slot = nf.capture_adapters(4, 96, 4, False)
        none = nf.run(slot, inp, np.full(4, -1, np.int32))
        assert np.array_equal(nf.run(slot, inp)[0], none[0])
        ad = make_adapter(cfg, 9, 16)
        nf.set_adapter(0, ad, 0.0)
        nf.set_adapter(2, ad, 1.0)
        assert np.array_equal(nf.run(slot, inp, np.zeros(4, np.int32))[0], none[0])   # scaling 0
        assert np.array_equal(nf.run(slot, inp, np.ones(4, np.int32))[0], none[0])    # never set
        mixed = nf.run(slot, inp, np.array([2, -1, 2, -1], np.int32))
        assert not np.array_equal(mixed[0][0], none[0][0])
        # question 1 shares tiles with its neighbours' adapters and is untouched by them
        assert np.array_equal(mixed[0][1], none[0][1]) and np.array_equal(mixed[1][1], none[1][1])
        nf.clear_adapter(2)
        assert np.array_equal(nf.run(slot, inp, np.array([2, -1, 2, -1], np.int32))[0], none[0])
        mm = inp["marker_mask"]
        assert np.abs(none[0][mm] - plain[0][mm]).max() <= TOL["bf16"]
        assert np.array_equal(nf.run(0, inp)[0], plain[0])  # the plain slot is what it was
        for bad in (np.array([3, -1, -1, -1], np.int32), np.array([-2, -1, -1, -1], np.int32)):
            with pytest.raises(RuntimeError, match="adapter"):
                nf.run(slot, inp, bad)
        with pytest.raises(RuntimeError, match="captured without adapters"):
            nf.run(0, inp, np.full(4, -1, np.int32))
        with pytest.raises(RuntimeError, match="already enabled"):
            nf.enable_adapters(2, 8)
        ms = nf.replay_device(slot, 2, 15) if nf.run(slot, inp) else None
        assert (ms > 0).all() and nf.kernel_count(slot) > 0
    finally:
        nf.close()
    nf = NativeForward(0, cfg, w, "nvfp4", max_batch=2, max_options=4)
    try:
        with pytest.raises(RuntimeError, match="NVFP4"):
            nf.enable_adapters(2, 8)
        with pytest.raises(RuntimeError, match="not enabled"):
            nf.capture_adapters(2, 64, 4, False)
    finally:
        nf.close()


def test_engine_lanes_tables_and_changes_of_adapters():
    cfg = TINY
    w = seeded_weights(cfg, seed=7)
    ads = {nm: (make_adapter(cfg, s, 16), 2.0) for s, nm in ((1, "a"), (2, "b"), (3, "c"))}
    items = synthetic_items([64, 40, 64, 33], ["choice", "noul", "score", "noul"], seed=4, vocab=cfg.vocab)

    def request(*names):
        return request_from_items([dict(it, adapter=n) for it, n in zip(items, names)])

    with B200Engine(config=cfg, weights=w, device=0, max_questions=8, max_options=4, lanes=2, token_tables=True,
                    adapters=2, adapter_rank=16, sequence_buckets=(64,)) as eng:
        plain = eng.run_prepared(request(None, None, None, None))[0]
        eng.load_adapter("a", *ads["a"])
        eng.load_adapter("b", *ads["b"])
        ref = {}
        for names in (("a", "b", None, "a"), ("b", None, "b", "b"), (None, "a", "a", None)):
            chosen = [ads[n] if n else None for n in names]
            inp = pack(items, 4, 64, 4, cfg.pad_token_id)
            want = AdaptedOracle(w, cfg, chosen).forward(**inp)[0]
            got, _, meta = eng.run_prepared(request(*names))
            ref[names] = got
            assert np.abs(got - want)[inp["marker_mask"]].max() <= TOL["bf16"]
        assert np.array_equal(eng.run_prepared(request(None, None, None, None))[0], plain)
        # both lanes at once, each with its own mix
        wrong = []

        def serve(names):
            for _ in range(20):
                if not np.array_equal(eng.run_prepared(request(*names))[0], ref[names]):
                    wrong.append(names)

        threads = [threading.Thread(target=serve, args=(n,)) for n in ref]
        for t in threads:
            t.start()
        # replaced while they run: the same adapter, so no result may change
        for _ in range(3):
            eng.load_adapter("b", *ads["b"])
        for t in threads:
            t.join()
        assert not wrong
        eng.unload_adapter("a")
        with pytest.raises(ValueError):
            eng.run_prepared(request("a", None, None, None))
        eng.load_adapter("c", *ads["c"])
        got = eng.run_prepared(request("c", "b", "c", None))[0]
        want = AdaptedOracle(w, cfg, [ads["c"], ads["b"], ads["c"], None]).forward(**inp)[0]
        assert np.abs(got - want)[inp["marker_mask"]].max() <= TOL["bf16"]
