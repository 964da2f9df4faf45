"""The engine with adapters whose effect on the answers is several times what its
precision may be off by: an engine that left them out, or took another question's,
would not pass.  (The other adapter tests use small ones, near the weights' size.)"""
import threading

import numpy as np
import pytest

from laya_b200.config import TINY
from laya_b200.engine import B200Engine, request_from_items
from laya_b200.weights import seeded_weights
from laya_b200.workload import pack, synthetic_items
from oracle import laya_oracle as O
from test_gpu_adapters import TOL, WIDE, AdaptedOracle, compare, make_adapter

pytestmark = pytest.mark.gpu


def large(cfg, size=0.1):
    return {"a": (make_adapter(cfg, 1, 16, size=size), 2.0), "b": (make_adapter(cfg, 2, 7, size=size), 4.0)}


@pytest.mark.parametrize("lengths, batch, seq, names", [
    ([64], 1, 64, ["a"]), ([20], 1, 32, ["b"]), ([96, 50, 70, 96], 4, 96, ["a", "b", None, "a"]),
    ([512, 300, 64, 90, 400], 8, 512, ["b", None, "a", "a", "b"])])
@pytest.mark.parametrize("precision", ["bf16", "fp8"])
def test_large_adapters(lengths, batch, seq, names, precision):
    w = seeded_weights(TINY, seed=5)
    got, ref, plain, mm = compare(TINY, precision, w, large(TINY), lengths, batch, seq, names)
    err, moved = np.abs(got[0] - ref[0])[mm].max(), np.abs(plain[0] - ref[0])[mm].max()
    print(f"large adapters {precision} {batch}x{seq}: logits {err:.3e}, adapters move them {moved:.3e}")
    assert moved > 1.5 * TOL[precision]  # by the oracle alone
    assert err <= TOL[precision] and err < moved / 4


@pytest.mark.parametrize("precision", ["bf16", "fp8"])
def test_large_adapters_on_wide_tiles(precision):
    w = seeded_weights(WIDE, seed=8)
    lengths = [256, 200, 256, 64, 31, 256, 180, 256, 100, 256]
    names = ["a", "b", None, "a", "a", "b", None, "b", "a", "a"]
    got, ref, plain, mm = compare(WIDE, precision, w, large(WIDE, 0.05), lengths, 16, 256, names, slots=2, rank=64)
    err, moved = np.abs(got[0] - ref[0])[mm].max(), np.abs(plain[0] - ref[0])[mm].max()
    print(f"large adapters {precision} wide: logits {err:.3e}, adapters move them {moved:.3e}")
    assert moved > 1.5 * TOL[precision]
    assert err <= TOL[precision] and err < moved / 4


@pytest.mark.parametrize("precision", ["bf16", "fp8"])
def test_lanes_with_large_adapters(precision):
    cfg, ads = TINY, large(TINY)
    w = seeded_weights(cfg, seed=5)
    items = synthetic_items([64, 40, 64, 33], ["choice", "noul", "score", "noul"], seed=4, vocab=cfg.vocab)
    inp = pack(items, 4, 64, 4, cfg.pad_token_id)
    mm = inp["marker_mask"]
    plain = O.Oracle(w, cfg, precision).forward(**inp)[0]
    mixes = (("a", "b", None, "a"), ("b", None, "b", "b"), (None, "a", "a", None))
    with B200Engine(config=cfg, weights=w, device=0, max_questions=8, max_options=4, lanes=2, adapters=2,
                    adapter_rank=16, sequence_buckets=(64,), precision=precision) as eng:
        for nm, ad in ads.items():
            eng.load_adapter(nm, *ad)
        got = {}

        def serve(names):
            for _ in range(5):
                got.setdefault(names, []).append(eng.run_prepared(request_from_items(
                    [dict(it, adapter=n) for it, n in zip(items, names)]))[0])

        threads = [threading.Thread(target=serve, args=(n,)) for n in mixes]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    for names in mixes:
        ref = AdaptedOracle(w, cfg, [ads[n] if n else None for n in names], precision).forward(**inp)[0]
        err = max(np.abs(g - ref)[mm].max() for g in got[names])
        chosen = mm & np.array([n is not None for n in names])[:, None]
        moved = np.abs(plain - ref)[chosen].max()
        print(f"lanes {precision} {names}: logits {err:.3e}, adapters move them {moved:.3e}")
        assert moved > 1.5 * TOL[precision]
        assert err <= TOL[precision] and err < moved / 4
        assert all(np.array_equal(g, got[names][0]) for g in got[names])
