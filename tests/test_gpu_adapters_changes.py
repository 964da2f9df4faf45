"""Adapters loaded and cleared while another engine on the GPU captures its graphs."""
import threading

import numpy as np
import pytest

from laya_b200.config import TINY
from laya_b200.engine import B200Engine, request_from_items
from laya_b200.weights import seeded_weights
from laya_b200.workload import synthetic_items
from test_gpu_adapters import make_adapter

pytestmark = pytest.mark.gpu


def test_changes_beside_another_engines_captures():
    w = seeded_weights(TINY, seed=3)
    ad = make_adapter(TINY, 1, 8)
    requests = [request_from_items(synthetic_items([n], ["noul"], seed=n, vocab=TINY.vocab)) for n in (30, 60)]
    kw = dict(config=TINY, weights=w, device=0, max_questions=2, max_options=4, sequence_buckets=(32, 64))
    with B200Engine(adapters=2, adapter_rank=8, **kw) as a, B200Engine(max_graphs=1, **kw) as b:
        refs = [b.run_prepared(r)[0] for r in requests]
        stop, failed = threading.Event(), []

        def change():
            try:
                while not stop.is_set():
                    a.load_adapter("x", ad)
                    a.unload_adapter("x")
            except Exception as e:
                failed.append(e)

        t = threading.Thread(target=change)
        t.start()
        try:
            for i in range(150):  # one graph is kept: every request captures
                out, _, meta = b.run_prepared(requests[i % 2])
                assert meta["graph_miss"] and np.array_equal(out, refs[i % 2])
        finally:
            stop.set()
            t.join()
        assert not failed, failed
